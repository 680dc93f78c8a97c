// Many query rows against cache rows on tcgen05: prompts over their own rows, and a prefix for all the sequences
// that share it.
//
// An item is up to 256 query rows of one key head (two 128-row tiles) and the cache rows that they see, in blocks of
// 128; every thread block gets the same number of units (128 cache rows against both tiles) and goes through them item
// by item.  Per block of cache rows and tile:
//   S = Q K^T (128 x 128, TMEM)  ->  P = 2^(S c - m), rounded to bf16 into the columns S came from  ->  O += P V (TMEM)
// A thread owns a query row: maximum and sum need no exchange, and O is scaled only when a row's maximum has moved
// by more than 2^8.  The two tiles take turns: while one's softmax runs, the other's products do.  Where an item has
// one tile only (a prefix under few tokens), the two sides take every other block of cache rows, and join at the end.
//
// Warps: 0 loads K and V by TMA into a ring of 32 KB buffers, 1 issues the products, 4-7 and 8-11 are the two sides.
// With `mass` the queries' rounding remainder multiplies too (S += Qlo K^T), as sums of weights are kept in 32 bits; without it the
// query is rounded to bf16 as P is, each by at most 2^-8, in no common direction.
#include <cuda.h>
#include "cached_attention.cuh"
#include "launchers.h"
#include "packed.cuh"
#include "sm100.cuh"
#include "tmap.h"
#include "umma.cuh"

using namespace ahb;
using namespace ahb::cattn;
using sm100::mbar_arrive;
using sm100::mbar_expect_tx;
using sm100::mbar_init;
using sm100::mbar_wait;
using sm100::smem_u32;
using sm100::tc_fence_after;
using sm100::tc_fence_before;

namespace {

constexpr int NTHR = 384;
constexpr uint32_t BUF = 32 * 1024;  // one block of K or V (or a tile of queries), two 64-channel slabs of 128 rows
constexpr int COL_O = 256;           // TMEM columns: S and P of the sides at 0 and 128, O at 256 and 384

template <bool EXACT>
constexpr int ring() { return EXACT ? 3 : 5; }
template <bool EXACT>
constexpr size_t smem_bytes() { return (size_t)BUF * (ring<EXACT>() + (EXACT ? 4 : 2)) + 1024 + 2048; }

struct Item {
  int pre, h, r0, rows, blocks, ks, ke;  // units ks .. ke of the item
  bool two, whole;                       // two tiles; all of the item's units
  bool late;                             // the item began before this block's units
  Group g;
  // blocks of cache rows of side w in these units, and the j-th of them
  AHB_DEVICE int count(int w) const { return (two ? ke : min(ke, (blocks - w + 1) >> 1)) - ks; }
  AHB_DEVICE int block(int w, int j) const { return two ? ks + j : 2 * (ks + j) + w; }
};

// The item that holds unit u, as far as this block's units go; moves u behind it.
AHB_DEVICE Item next_item(const Args& a, int64_t& u, int64_t u_first, int64_t u_end) {
  const int64_t *own = a.sums[TILES], *runs = own + a.B + 1;
  const int64_t n_own = own[a.B];
  Item it;
  it.pre = u >= n_own;
  const int64_t* sums = it.pre ? runs : own;
  const int64_t v = it.pre ? u - n_own : u;
  const int i = find_group(sums, a.B, v);
  it.g = a.groups[it.pre ? a.B + i : i];
  const int64_t base = sums[i], per_head = (sums[i + 1] - base) / a.Hk;
  it.h = (int)((v - base) / per_head);
  int rest = (int)(v - base - it.h * per_head), rt = 0;
  TileItem t = tile_item(a, it.g, 0);
  while (rest >= t.units) {
    rest -= t.units;
    t = tile_item(a, it.g, ++rt);
  }
  it.r0 = rt * 2 * TQ;
  it.rows = t.rows;
  it.blocks = t.blocks;
  it.two = t.rows > TQ;
  it.ks = rest;
  it.ke = (int)min((int64_t)t.units, rest + (u_end - u));
  it.whole = it.ks == 0 && it.ke == t.units;
  it.late = u - rest < u_first;
  u += it.ke - it.ks;
  return it;
}

// The order in which blocks of K and V go through the ring: the sides' first K, then for every step and side V and the next
// step's K.  With two tiles both sides read the same ones.  f(is V, side, step).
template <class F>
AHB_DEVICE void in_order(const Item& it, F&& f) {
  const int n0 = it.count(0), n1 = it.two ? 0 : it.count(1);
  f(false, 0, 0);
  if (n1 > 0) f(false, 1, 0);
  for (int j = 0; j < n0; ++j) {
    f(true, 0, j);
    if (j + 1 < n0) f(false, 0, j + 1);
    if (j < n1) f(true, 1, j);
    if (j + 1 < n1) f(false, 1, j + 1);
  }
}

AHB_DEVICE void umma_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of the warp's lanes, not waited for; `arrived` after tmem_wait keeps their uses behind it
AHB_DEVICE void tmem_get32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
AHB_DEVICE void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
template <int N>
AHB_DEVICE void arrived(float* v) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
AHB_DEVICE void tmem_put32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
AHB_DEVICE void tmem_put16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
AHB_DEVICE void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// named barriers of the softmax warps: 1 both sides
AHB_DEVICE void sides_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D, bool EXACT>
__global__ void __launch_bounds__(NTHR, 1)
    ca_tiles(const Args a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  constexpr int NB = ring<EXACT>(), SLABS = (D + 63) / 64, DC = (D + 31) / 32;
  constexpr uint32_t SLAB = TK * 128, LOAD = SLABS * SLAB;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = smem;                               // tiles of queries (EXACT: rounded ones, then remainders)
  unsigned char* kv = smem + BUF * (EXACT ? 4 : 2);       // the ring
  uint64_t* bars = reinterpret_cast<uint64_t*>(kv + BUF * NB);
  uint64_t *kv_full = bars, *kv_empty = bars + NB, *q_full = bars + 2 * NB, *s_full = q_full + 2, *p_full = s_full + 2,
           *o_full = p_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* other = reinterpret_cast<float2*>(tmem_slot + 4);  // the second side's maximum and sum, row by row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t* sums = a.sums[TILES];
  const int64_t all = sums[a.B] + sums[2 * a.B + 1], share = share_of(all, a.blocks);
  const int64_t u_first = (int64_t)blockIdx.x * share, u_end = min(u_first + share, all);
  if (u_first >= u_end) return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 128);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(o_full + i, 1);
    }
    *abort_flag = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 2) sm100::tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int64_t u = u_first;
  // registers: 3 x 168 at the launch = 88 + 2 x 208
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {  // ------------------------------------------------ loads
    uint32_t n = 0;
    bool ok = true;
    while (u < u_end && ok) {
      const Item it = next_item(a, u, u_first, u_end);
      if (lane == 0) {
        const int plane = it.g.slot * a.Hk + it.h;
        in_order(it, [&](bool is_v, int w, int j) {
          if (!ok) return;
          const uint32_t b = n % NB;
          if (n >= NB && !mbar_wait(kv_empty + b, ((n / NB) & 1) ^ 1, abort_flag, a.err, 61)) {
            ok = false;
            return;
          }
          mbar_expect_tx(kv_full + b, LOAD);
          const int row = it.block(w, j) * TK;
#pragma unroll
          for (int s = 0; s < SLABS; ++s)
            umma::tma_load_3d(kv + b * BUF + s * SLAB, is_v ? &mv : &mk, kv_full + b, 64 * s, row, plane);
          ++n;
        });
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    if (lane == 0)  // copies in flight end before the block does
      for (uint32_t i = n > NB ? n - NB : 0; i < n; ++i) umma::wait_bar(kv_full + i % NB, (i / NB) & 1, a.err, 62);
  } else if (warp == 1) {  // ----------------------------------------- products
    constexpr uint32_t ID_S = sm100::idesc_bf16(TQ, TK, false, false), ID_O = sm100::idesc_bf16(TQ, D, false, true);
    uint32_t n = 0, np[2] = {0, 0}, nq[2] = {0, 0};
    bool ok = true;
    while (u < u_end && ok) {
      const Item it = next_item(a, u, u_first, u_end);
      if (lane == 0) {
        const int cnt[2] = {it.count(0), it.count(1)};
        // the buffer that comes next in the ring, once it is filled
        auto next = [&]() {
          const uint32_t b = n % NB;
          ok = ok && mbar_wait(kv_full + b, (n / NB) & 1, abort_flag, a.err, 63);
          ++n;
          return b;
        };
        auto wait_q = [&](int w) {
          ok = ok && mbar_wait(q_full + w, nq[w] & 1, abort_flag, a.err, 64);
          ++nq[w];
        };
        auto score = [&](int w, uint32_t b) {
          if (!ok) return;
          const uint32_t q = smem_u32(qs) + (it.two ? w : 0) * BUF, k = smem_u32(kv) + b * BUF;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            sm100::umma_bf16(tmem + 128 * w, umma::kdesc(q, TQ, s), umma::kdesc(k, TK, s), ID_S, s > 0);
          if (EXACT) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
              sm100::umma_bf16(tmem + 128 * w, umma::kdesc(q + 2 * BUF, TQ, s), umma::kdesc(k, TK, s), ID_S, 1);
          }
          sm100::umma_commit(s_full + w);
        };
        wait_q(0);
        if (it.two) wait_q(1);
        uint32_t kb = next();
        score(0, kb);
        if (!it.two) sm100::umma_commit(kv_empty + kb);
        if (cnt[1] > 0) {
          if (!it.two) kb = next();
          score(1, kb);
          sm100::umma_commit(kv_empty + kb);
        } else if (it.two) {
          sm100::umma_commit(kv_empty + kb);
        }
        for (int j = 0; j < cnt[0] && ok; ++j) {
          uint32_t vb = 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (j >= cnt[w] || !ok) continue;
            if (w == 0 || !it.two) vb = next();
            ok = ok && mbar_wait(p_full + w, np[w] & 1, abort_flag, a.err, 65);
            ++np[w];
            if (!ok) continue;
            tc_fence_after();
            const uint32_t v = smem_u32(kv) + vb * BUF;
#pragma unroll
            for (int s = 0; s < TK / 16; ++s)
              umma_ts(tmem + COL_O + 128 * w, tmem + 128 * w + 8 * s, umma::mndesc(v, TK, s), ID_O, j > 0 || s > 0);
            if (w == 1 || !it.two) sm100::umma_commit(kv_empty + vb);
            if (j + 1 < cnt[w]) {
              if (w == 0 || !it.two) kb = next();
              score(w, kb);
              if (ok && (w == 1 || !it.two)) sm100::umma_commit(kv_empty + kb);
            } else {
              sm100::umma_commit(o_full + w);
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
  }
  } else {  // ------------------------------------------ softmax: side w, a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int w = (warp - 4) >> 2, quarter = warp & 3, row = 32 * quarter + lane, G = a.H / a.Hk;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const uint32_t t_s = tmem + lanes + 128 * w, t_o = tmem + lanes + COL_O + 128 * w;
    uint32_t n = 0, ns = 0, no = 0;  // buffers through the ring, scores and results seen
    bool ok = true;
    // a whole warp's wait; after one that ran out the items are only counted, so that both sides meet at their barriers
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag, a.err, code));
    };
    while (u < u_end) {
      const Item it = next_item(a, u, u_first, u_end);
      const int r = it.r0 + row + (it.two ? TQ * w : 0), tt = r / G;
      const bool mine = r < it.r0 + it.rows;
      const int64_t out = mine ? (int64_t)(it.g.row0 + tt) * a.H + it.h * G + (r - tt * G) : -1;
      if (w == 0 || it.two) {  // the tile of queries; its last readers have been waited for
        const uint4* src = reinterpret_cast<const uint4*>(a.qw + out * 2 * D);
        const uint32_t dst = smem_u32(qs) + w * BUF;
#pragma unroll
        for (int x = 0; x < (EXACT ? 2 : 1); ++x)
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint4 q = mine ? src[x * (D / 8) + c] : make_uint4(0, 0, 0, 0);
            umma::st_shared16(dst + 2 * x * BUF + umma::sw_off16(TQ, row, 8 * c), q.x, q.y, q.z, q.w);
          }
        umma::fence_async_smem();
        mbar_arrive(q_full + w);
      }
      const int cnt = it.count(w), last = min(it.g.keys - 1, it.g.before + (mine ? tt : 0));
      // Cache rows behind the last one are made zero among the last block's values, as 0 times infinity is none; that
      // block is a side's last one, and its values are last or last but one in the ring's order
      const int n0 = it.count(0), n1 = it.two ? 0 : it.count(1);
      n += 2 * (n0 + n1);
      const bool tail = cnt > 0 && (it.block(w, cnt - 1) + 1) * TK > it.g.keys && !(it.two && w == 1);
      const uint32_t tail_buf = n - (it.two || (n1 == n0) == (w == 1) ? 1 : 2);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < cnt && ok; ++j) {
        const int k0 = it.block(w, j) * TK;
        ok = wait(s_full + w, ns, 66);
        ++ns;
        if (!ok) break;
        tc_fence_after();
        float s[TK];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_get32(t_s + 32 * c, s + 32 * c);
        tmem_wait();
        arrived<TK>(s);
        if (__any_sync(0xffffffffu, k0 + TK - 1 > last)) {
#pragma unroll
          for (int c = 0; c < TK; ++c) s[c] = k0 + c <= last ? s[c] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < TK; c += 4)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[c + e]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
        if (__any_sync(0xffffffffu, top > m + SLACK)) {
          const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : ex2(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < DC; ++c) {
              float o[32];
              tmem_get32(t_o + 32 * c, o);
              tmem_wait();
              arrived<32>(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
              tmem_put32(t_o + 32 * c, reinterpret_cast<uint32_t*>(o));
            }
          }
        }
        const float2 neg = both(m == -INFINITY ? 0.f : -m), scale = both(a.scale2);
        float2 sum = both(0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = fma2(make_float2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), scale, neg);
            const float2 y = make_float2(ex2(x.x), ex2(x.y));
            sum = add2(sum, y);
            p[e] = umma::pack_bf2(y.x, y.y);
          }
          tmem_put16(t_s + 16 * c, p);
        }
        l += sum.x + sum.y;
        tmem_put_wait();
        if (tail && j == cnt - 1) {
          ok = wait(kv_full + tail_buf % NB, tail_buf / NB, 67);
          if (k0 + row >= it.g.keys) {
            const uint32_t at = smem_u32(kv) + (tail_buf % NB) * BUF + row * 128;
#pragma unroll
            for (int x = 0; x < SLABS; ++x)
#pragma unroll
              for (int c = 0; c < 8; ++c) umma::st_shared16(at + x * SLAB + 16 * c, 0, 0, 0, 0);
          }
          umma::fence_async_smem();
        }
        tc_fence_before();
        mbar_arrive(p_full + w);
      }
      if (cnt > 0 && ok) {
        ok = wait(o_full + w, no, 68);
        ++no;
        tc_fence_after();
      }
      // every thread comes to the barriers, whatever its waits said
      float f0 = 1.f, f1 = 0.f;
      if (!it.two) {
        if (w == 1) other[row] = make_float2(m, l);
        sides_sync();
        if (w == 0) {
          const float2 b = other[row];
          if (b.x != -INFINITY) {
            const float mn = fmaxf(m, b.x);
            f0 = m == -INFINITY ? 0.f : ex2(m - mn);
            f1 = ex2(b.x - mn);
            l = l * f0 + b.y * f1;
            m = mn;
          }
        }
      }
      if (ok && (w == 0 || it.two)) {
        const bool final = it.whole && !a.full, join = !it.two && it.count(1) > 0;
        const float inv = final ? 1.f / l : 1.f;
        float* y = nullptr;
        if (!final)
          y = it.whole ? a.full + ((int64_t)(it.pre ? a.T : 0) * a.H + out) * (D + 2)
                       : a.tile_part + ((2 * (int64_t)blockIdx.x + (it.late ? 0 : 1)) * 2 * TQ + r - it.r0) * (D + 2);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          float o[32];
          tmem_get32(t_o + 32 * c, o);
          if (join) {
            float b[32];
            tmem_get32(t_o + 128 + 32 * c, b);
            tmem_wait();
            arrived<32>(o);
            arrived<32>(b);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = o[e] * f0 + (f1 > 0.f ? b[e] * f1 : 0.f);
          } else {
            tmem_wait();
            arrived<32>(o);
          }
          if (mine && final) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = o[e + k] * inv;
              *reinterpret_cast<uint4*>(a.o + out * D + 32 * c + e) = umma::pack8(x);
            }
          } else if (mine) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) *reinterpret_cast<float2*>(y + 32 * c + e) = make_float2(o[e], o[e + 1]);
          }
          __syncwarp();
        }
        if (mine) {
          if (!final) *reinterpret_cast<float2*>(y + D) = make_float2(m, l);
          else if (a.lse) a.lse[out] = m + log2f(l);
        }
      }
      tc_fence_before();
      if (!it.two) sides_sync();  // the second side's O has been read
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) sm100::tmem_dealloc(tmem, 512);
}

// bf16 caches (S Hk, M, D): boxes of 64 channels and 128 rows of one slot's head, rows past M as zeros
int map_cache(CUtensorMap* m, const void* p, const Args& a) {
  TmapEncodeFn fn = tmap_encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.M, (cuuint64_t)a.S * a.Hk};
  cuuint64_t strides[2] = {(cuuint64_t)a.D * 2, (cuuint64_t)a.M * a.D * 2};
  cuuint32_t box[3] = {64, TK, 1}, es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : -2;
}

template <int D, bool EXACT>
int launch_one(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  constexpr int bytes = (int)smem_bytes<EXACT>();
  if (cudaFuncSetAttribute(ca_tiles<D, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -3;
  ca_tiles<D, EXACT><<<a.blocks, NTHR, bytes, st>>>(a, mk, mv);
  return 0;
}

template <int D>
int launch_dim(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  return a.mass ? launch_one<D, true>(a, mk, mv, st) : launch_one<D, false>(a, mk, mv, st);
}

}  // namespace

int ahb::cattn::launch_tiles(const Args& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  if (map_cache(&mk, a.kc, a) || map_cache(&mv, a.vc, a)) return -2;
  switch (a.D) {
    case 64: return launch_dim<64>(a, mk, mv, st);
    case 96: return launch_dim<96>(a, mk, mv, st);
    default: return launch_dim<128>(a, mk, mv, st);
  }
}
