// Many query rows against cache rows on tcgen05: prompts over their own rows, and a prefix for all the sequences
// that share it.
//
// An item is up to 256 query rows of one key head (two 128-row tiles) and the cache rows that they see, in blocks of
// 64; every thread block gets the same number of units (64 cache rows against both tiles) and goes through them item
// by item.  Per block of cache rows and tile:
//   S = Q K^T (128 x 64, TMEM)  ->  P = 2^(S c - m), rounded to bf16 (TMEM)  ->  O += P V (TMEM)
// A thread owns a query row: maximum and sum need no exchange, and O is scaled only when a row's maximum has moved
// by more than 2^8.  The next S is made as soon as the softmax holds the last one in registers, P has two places of its own
// (products of different shapes do not wait for one another: S must not come to where P V still reads), and the two tiles'
// softmaxes share the exponential unit between them.  Where an item has
// one tile only (a prefix under few tokens), the two sides take every other block of cache rows, and join at the end.
//
// Queries are multiplied as rounded to bf16 and, in as many products more, what the rounding left of them: rounded alone they move
// every score by up to 2^-8 of its terms, and an output twice as far as its own rounding does (a prompt of 8192 tokens then takes
// 402 us instead of 508).  P is rounded to bf16, each weight by at most 2^-8 in no common direction, which moves an output
// about as far as its own rounding; the sums of weights are of those before it, in 32 bits.
//
// Warps: 0 loads K and V by TMA into a ring of three 32 KB buffers, 3 the tiles of queries, 1 and 2 issue the two sides' products
// (one thread for both spent as long on its waits and commits as the tensor cores on the products, so a prompt of 8192 tokens
// took twice as long), 4-7 and 8-11 are the sides' softmaxes.
// A step of 64 cache rows and both tiles takes 2700 cycles.  The products need 2080 of them, as S (N = 64) is bound by what a
// product reads from shared memory, 49 cycles where the tensor cores need 32; the exponentials need 1020.  (8192 tokens of 16 heads
// of 128: 275 GFLOP in 418 us, the products of the remainders not counted.)  A second S buffer a side, with P in its place
// and S waiting for P V, was slower (558 us in all): it brings the products into one order with the softmaxes.
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
constexpr uint32_t QBUF = 32 * 1024;  // a tile of queries: two 64-channel slabs of 128 rows
constexpr uint32_t HALF = 16 * 1024;  // a block of K or V: two 64-channel slabs of 64 rows
constexpr uint32_t BUF = 2 * HALF;    // what a step multiplies: the K of its S, the V of its P
constexpr int COL_P = 64, COL_O = 256;  // TMEM columns: side w's S at 128 w, its P buffer b at 128 w + 64 + 32 b, its O at 256 + 128 w

constexpr uint32_t STAGE = 4 * 1024;  // a softmax warp's results on their way out, where the queries were
constexpr int NB = 3;                 // buffers of the ring
constexpr size_t SMEM_BYTES = (size_t)BUF * NB + QBUF * 4 + 1024 + 2048;  // all that a block can have

struct Item {
  int pre, h, r0, rows, blocks, ks, ke;  // units ks .. ke of the item
  bool two, whole;                       // two tiles; all of the item's units
  int64_t u_last;                        // the item's last unit
  bool late;                             // its first block of cache rows came before this thread block's units
  Group g;
  // blocks of cache rows of side w in these units, and the j-th of them
  AHB_DEVICE int count(int w) const { return (two ? ke : min(ke, (blocks - w + 1) >> 1)) - ks; }
  AHB_DEVICE int block(int w, int j) const { return two ? ks + j : 2 * (ks + j) + w; }
};

// Where a thread block is in its units.
struct Place {
  int64_t u, u_first, u_end;
  int x, h, rt, at;  // group, key head, 256-row tile and the unit within it; x < 0: not looked up yet
};

// The next item, as far as this block's units go (the last one may be without a block of cache rows: ke <= ks); moves the
// place behind it.  A whole warp calls it.
AHB_DEVICE Item next_item(const Args& a, Place& p) {
  const int64_t *own = a.sums[TILES], *runs = own + a.B + 1;
  const int64_t n_own = own[a.B];
  Item it;
  TileItem t;
  bool found = false;
  if (p.x >= 0) {  // on from the last one: its next tile, its next head
    it.g = a.groups[p.x];
    if (++p.rt == row_tiles(a, it.g)) p.rt = 0, ++p.h;
    p.at = 0;
    found = p.h < a.Hk;
  }
  if (!found) {
    const bool pre = p.u >= n_own;
    const int64_t *sums = pre ? runs : own, v = pre ? p.u - n_own : p.u;
    const int i = find_group(sums, a.B, v), lane = threadIdx.x & 31;
    p.x = pre ? a.B + i : i;
    it.g = a.groups[p.x];
    const int64_t base = sums[i];
    p.h = (int)div64(v - base, it.g.per_head);
    int64_t rest = v - base - p.h * it.g.per_head;
    const int tiles = row_tiles(a, it.g);
    for (p.rt = 0;; p.rt += 32) {  // 32 tiles at a time
      const int64_t mine = p.rt + lane < tiles ? tile_item(a, it.g, p.rt + lane).units : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, upto > rest);
      if (behind) {
        const int k = __ffs(behind) - 1;
        rest -= __shfl_sync(0xffffffffu, upto - mine, k);
        p.rt += k;
        break;
      }
      rest -= __shfl_sync(0xffffffffu, upto, 31);
    }
    p.at = (int)rest;
  }
  t = tile_item(a, it.g, p.rt);
  it.pre = p.x >= a.B;
  it.h = p.h;
  it.r0 = p.rt * 2 * a.tile_rows;
  it.rows = t.rows;
  it.blocks = t.blocks;
  it.two = t.rows > a.tile_rows;
  const int to = (int)min((int64_t)t.units, p.at + (p.u_end - p.u));
  it.ks = max(p.at - ITEM_COST, 0);
  it.ke = to - ITEM_COST;
  it.whole = it.ks == 0 && to == t.units;
  it.late = p.u - p.at + ITEM_COST < p.u_first;
  it.u_last = p.u - p.at + t.units - 1;
  p.u += to - p.at;
  return it;
}

// A side's steps are j = -2 .. n - 1 for n blocks: step j makes S(j + 2) and multiplies P(j) V(j), where there are such, once
// the softmax has taken S(j + 1) into registers, with P(j) behind it.  What a step reads is one filling of the ring: K(j + 2)
// and V(j); with two tiles both sides read the same one, else side 0's and side 1's take turns.
AHB_DEVICE bool has_step(int j, int n) { return (j >= 0 && j < n) || (j < 0 && j + 2 < n); }
AHB_DEVICE int fillings(int n) { return n > 1 ? n + 2 : 2 * n; }

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
AHB_DEVICE void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 4-D TMA tile load (no multicast)
AHB_DEVICE void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// A warp's 32 rows of B bytes (64 or 128), a row a thread, through shared memory, so that every row leaves in whole
// 32-byte sectors: thread `lane` hands out chunk lane % C of rows lane / C, lane / C + R, ..  place[i]: which row of `out`,
// `stride` bytes apart, the i-th of those is; negative for none.
template <int B>
struct RowsOut {
  static constexpr int C = B / 16, R = 32 / C;  // chunks a row, rows at a time
  int place[C];
  AHB_DEVICE RowsOut(int mine) {
#pragma unroll
    for (int i = 0; i < C; ++i) place[i] = __shfl_sync(0xffffffffu, mine, i * R + (threadIdx.x & 31) / C);
  }
  static AHB_DEVICE int at(int row, int c) { return row * B + ((B == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4); }
  AHB_DEVICE void write(unsigned char* stage, const uint4* v, unsigned char* out, int stride) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(stage + at(lane, c)) = v[c];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (place[i] >= 0)
        *reinterpret_cast<uint4*>(out + (int64_t)place[i] * stride + 16 * (lane % C)) =
            *reinterpret_cast<const uint4*>(stage + at(i * R + lane / C, lane % C));
    __syncwarp();
  }
};

// named barriers of the softmax warps: 1 both sides
AHB_DEVICE void sides_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// ROUNDED: see Args::rounded
template <int D, bool ROUNDED>
__global__ void __launch_bounds__(NTHR, 1)
    ca_tiles(const Args a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
             const __grid_constant__ CUtensorMap mq) {
  next_may_start();
  after_previous();
  constexpr int SLABS = (D + 63) / 64, DC = (D + 31) / 32;
  constexpr uint32_t SLAB = TK * 128, LOAD = SLABS * SLAB;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = smem;             // two tiles of rounded queries, then their remainders
  unsigned char* kv = smem + QBUF * 4;  // the ring
  uint64_t* bars = reinterpret_cast<uint64_t*>(kv + BUF * NB);
  // of side w: its steps are done (at 2 w, by turns), S is there, the softmax has taken it, with the P before it
  uint64_t *kv_full = bars, *kv_empty = bars + NB, *q_full = bars + 2 * NB, *q_empty = q_full + 2, *done = q_empty + 2, *s_full = done + 4,
           *taken = s_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* other = reinterpret_cast<float2*>(tmem_slot + 4);  // the second side's maximum and sum, row by row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t* sums = a.sums[TILES];
  const int64_t all = sums[a.B] + sums[2 * a.B + 1], share = share_of(all, a.blocks);
  Place at;
  at.u_first = at.u = (int64_t)blockIdx.x * share;
  at.u_end = min(at.u_first + share, all);
  at.x = -1;
  if (threadIdx.x == 0) a.shared_items[blockIdx.x].rows = 0;
  if (at.u >= at.u_end) return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 2);  // both sides'
    }
    for (int i = 0; i < 4; ++i) mbar_init(done + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(taken + i, 4);  // a side's warps
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 4);  // the warps whose results went through it
    }
    *abort_flag = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 3) sm100::tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // registers: 3 x 168 at the launch = 88 + 2 x 208
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {  // ------------------------------------------------ loads
    uint32_t n = 0;
    bool ok = true;
    while (at.u < at.u_end && ok) {
      const Item it = next_item(a, at);
      if (it.ke <= it.ks) break;
      if (lane == 0) {
        const int plane = it.g.slot * a.Hk + it.h;
        const int n0 = it.count(0), n1 = it.two ? 0 : it.count(1);
        for (int j = -2; j < n0; ++j)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int cnt = w ? n1 : n0;
            if (!has_step(j, cnt) || !ok) continue;
            const uint32_t b = n % NB;
            if (n >= NB && !mbar_wait(kv_empty + b, ((n / NB) & 1) ^ 1, abort_flag, a.err, 61)) {
              ok = false;
              continue;
            }
            const bool k = j + 2 < cnt, v = j >= 0;
            mbar_expect_tx(kv_full + b, (k ? LOAD : 0) + (v ? LOAD : 0));
#pragma unroll
            for (int s = 0; s < SLABS; ++s) {
              if (v) umma::tma_load_3d(kv + b * BUF + HALF + s * SLAB, &mv, kv_full + b, 64 * s, it.block(w, j) * TK, plane);
              if (k) umma::tma_load_3d(kv + b * BUF + s * SLAB, &mk, kv_full + b, 64 * s, it.block(w, j + 2) * TK, plane);
            }
            ++n;
          }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    if (lane == 0)  // copies in flight end before the block does
      for (uint32_t i = n > NB ? n - NB : 0; i < n; ++i) umma::wait_bar(kv_full + i % NB, (i / NB) & 1, a.err, 62);
  } else if (warp < 3) {  // ------------------------------------------ products of side w
    constexpr uint32_t ID_S = sm100::idesc_bf16(TQ, TK, false, false), ID_O = sm100::idesc_bf16(TQ, D, false, true);
    const int w = warp - 1;
    uint32_t n = 0, nd = 0, nt = 0, items = 0, twos = 0;  // fillings, steps, S taken, items, those of two tiles
    bool ok = true;
    while (at.u < at.u_end && ok) {
      const Item it = next_item(a, at);
      if (it.ke <= it.ks) break;
      if (lane == 0) {
        const int n0 = it.count(0), n1 = it.count(1), cnt = w ? n1 : n0, others = it.two ? 0 : w ? n0 : n1;
        // Both sides go through the whole ring in order, so that neither mistakes one filling of a buffer for another: what a
        // side does not use it gives back at once.
        auto pass = [&](int j) {
          if (!has_step(j, others)) return;
          ok = ok && mbar_wait(kv_full + n % NB, (n / NB) & 1, abort_flag, a.err, 63);
          if (ok) mbar_arrive(kv_empty + n % NB);
          ++n;
        };
        ok = ok && mbar_wait(q_full, items & 1, abort_flag, a.err, 64);
        if (it.two && w == 1) ok = ok && mbar_wait(q_full + 1, twos & 1, abort_flag, a.err, 64);
        ++items;
        twos += it.two;
        for (int j = -2; j < n0 && ok; ++j) {
          if (w == 1) pass(j);
          if (j < cnt && cnt > 0) {
            const bool some = has_step(j, cnt);
            const uint32_t b = n % NB, t_w = tmem + 128 * w;
            if (some) ok = ok && mbar_wait(kv_full + b, (n / NB) & 1, abort_flag, a.err, 63);
            if (j >= -1) {
              ok = ok && mbar_wait(taken + w, nt & 1, abort_flag, a.err, 65);
              ++nt;
            }
            if (!ok) break;
            uint32_t q = smem_u32(qs) + (it.two ? w : 0) * QBUF, k = smem_u32(kv) + b * BUF;
            asm volatile("" : "+r"(q), "+r"(k));  // descriptors made here, not kept over the loop in registers
            tc_fence_after();
            if (j + 2 < cnt) {
#pragma unroll
              for (int s = 0; s < D / 16; ++s) sm100::umma_bf16(t_w, umma::kdesc(q, TQ, s), umma::kdesc(k, TK, s), ID_S, s > 0);
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
                  sm100::umma_bf16(t_w, umma::kdesc(q + 2 * QBUF, TQ, s), umma::kdesc(k, TK, s), ID_S, 1);
              sm100::umma_commit(s_full + w);  // a completion is seen 500 cycles later: S is not to wait for P V
            }
            if (j >= 0) {
              const uint32_t t_p = t_w + COL_P + 32 * (j & 1);
#pragma unroll
              for (int s = 0; s < TK / 16; ++s)
                umma_ts(tmem + COL_O + 128 * w, t_p + 8 * s, umma::mndesc(k + HALF, TK, s), ID_O, j > 0 || s > 0);
            }
            sm100::umma_commit(done + 2 * w + ((nd + j) & 1));
            if (some) sm100::umma_commit(kv_empty + b);
            n += some;
          }
          if (w == 0) pass(j);
        }
        if (cnt > 0) nd += cnt + 2;
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
  } else if (warp == 3) {  // ----------------------------------------- tiles of queries
    uint32_t n[2] = {0, 0};
    bool ok = true;
    const int G = a.H / a.Hk;
    const uint32_t bytes = a.tile_rows * 128 * SLABS * 2;
    while (at.u < at.u_end && ok) {
      const Item it = next_item(a, at);
      if (it.ke <= it.ks) break;
      if (lane == 0) {
        const int t0 = it.g.row0 + per_group(it.r0, G), tokens = per_group(a.tile_rows, G);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (x && !it.two) break;
          if (n[x] > 0) ok = ok && mbar_wait(q_empty + x, (n[x] & 1) ^ 1, abort_flag, a.err, 70);
          if (!ok) break;
          mbar_expect_tx(q_full + x, bytes);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int s = 0; s < SLABS; ++s)
              tma_load_4d(qs + (x + 2 * e) * QBUF + s * TQ * 128, &mq, q_full + x, 64 * s, e, it.h * G, t0 + x * tokens);
          ++n[x];
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    if (lane == 0)
      for (int x = 0; x < 2; ++x)
        if (n[x] > 0) umma::wait_bar(q_full + x, (n[x] & 1) ^ 1, a.err, 71);
  }
  } else {  // --------------------------------------------------------- softmax: side w, a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int w = (warp - 4) >> 2, quarter = warp & 3, row = 32 * quarter + lane, G = a.H / a.Hk;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const uint32_t t_s = tmem + lanes + 128 * w, t_o = tmem + lanes + COL_O + 128 * w;
    uint32_t n = 0, nd = 0, ns = 0;  // fillings of the ring, steps of this side, its S
    bool ok = true;
    // a whole warp's wait; after one that ran out the items are only counted, so that both sides meet at their barriers
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag, a.err, code));
    };
    const float2 scale = both(a.scale2);
    while (at.u < at.u_end) {
      const Item it = next_item(a, at);
      if (it.ke <= it.ks) break;
      const int r_tile = it.r0 + (it.two ? a.tile_rows * w : 0);
      const int r = r_tile + row, tt = per_group(r, G);
      const bool mine = row < a.tile_rows && r < it.r0 + it.rows;
      const int64_t out = mine ? (int64_t)(it.g.row0 + tt) * a.H + it.h * G + (r - tt * G) : -1;
      const int cnt = it.count(w), last = min(it.g.keys - 1, it.g.before + (mine ? tt : 0));
      // Cache rows behind the last one are made zero among the last block's values, as 0 times infinity is none (by both
      // sides where both read them, each before its own products); that block is a side's last one, in the ring's last
      // filling, or the last but one if the other side's comes behind it
      const int n0 = it.count(0), n1 = it.two ? 0 : it.count(1);
      n += fillings(n0) + fillings(n1);
      const bool tail = cnt > 0 && (it.block(w, cnt - 1) + 1) * TK > it.g.keys;
      const uint32_t tail_buf = n - (it.two || (n1 == n0) == (w == 1) ? 1 : 2);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < cnt && ok; ++j, ++ns) {
        const int k0 = it.block(w, j) * TK;
        ok = wait(s_full + w, ns, 66);
        if (!ok) break;
        tc_fence_after();
        float s[TK];
        tmem_get32(t_s, s);
        tmem_get32(t_s + 32, s + 32);
        tmem_wait();
        arrived<TK>(s);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(taken + w);
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
        // what lies in a tile's rows of no query (its heads times tokens do not fill 128) decides nothing
        if (__any_sync(0xffffffffu, mine && top > m + SLACK)) {
          const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : ex2(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {
            ok = wait(done + 2 * w + ((nd + j + 1) & 1), (nd + j + 1) >> 1, 67);  // step j - 1: O has all before this block
            tc_fence_after();
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
        const float2 neg = both(m == -INFINITY ? 0.f : -m);
        float2 sum[2] = {both(0.f), both(0.f)};
        uint32_t p[TK / 2];
#pragma unroll
        for (int e = 0; e < TK / 2; ++e) {
          const float2 z = make_float2(s[2 * e], s[2 * e + 1]);
          // (packed products and sums came out as one fused operation again)
          const float2 x = ROUNDED ? make_float2(__fadd_rn(__fmul_rn(z.x, scale.x), neg.x), __fadd_rn(__fmul_rn(z.y, scale.y), neg.y))
                                   : fma2(z, scale, neg);
          const float2 y = make_float2(ex2(x.x), ex2(x.y));
          sum[e & 1] = add2(sum[e & 1], y);
          p[e] = umma::pack_bf2(y.x, y.y);
        }
        ok = wait(done + 2 * w + ((nd + j) & 1), (nd + j) >> 1, 67) && ok;  // step j - 2: P(j)'s place is free
        tc_fence_after();
        tmem_put32(t_s + COL_P + 32 * (j & 1), p);
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_put_wait();
      }
      if (cnt > 0) {
        // the last step but one: it has seen that the last S is taken, so that the last P is a new phase of that barrier; and what
        // filled the tail's buffer before has come and gone
        ok = ok && wait(done + 2 * w + ((nd + cnt) & 1), (nd + cnt) >> 1, 68);
        if (tail) {
          ok = ok && wait(kv_full + tail_buf % NB, tail_buf / NB, 68);
          if (row < TK && it.block(w, cnt - 1) * TK + row >= it.g.keys) {
            const uint32_t z = smem_u32(kv) + (tail_buf % NB) * BUF + HALF + row * 128;
#pragma unroll
            for (int x = 0; x < SLABS; ++x)
#pragma unroll
              for (int c = 0; c < 8; ++c) umma::st_shared16(z + x * SLAB + 16 * c, 0, 0, 0, 0);
          }
          umma::fence_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(taken + w);  // the last P
        ok = ok && wait(done + 2 * w + ((nd + cnt + 1) & 1), (nd + cnt + 1) >> 1, 69);  // the last step
        tc_fence_after();
        nd += cnt + 2;
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
        unsigned char* st = qs + (it.two ? w : 0) * QBUF + quarter * STAGE;  // no score of the item is to come
        auto result = [&](int c, float* o) {  // 32 channels of the row
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
        };
        if (final) {
          const RowsOut<64> rows((int)out);
          const float inv = 1.f / l;
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            float o[32];
            result(c, o);
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = o[8 * e + k] * inv;
              v[e] = umma::pack8(x);
            }
            rows.write(st, v, reinterpret_cast<unsigned char*>(a.o + 32 * c), D * 2);
          }
          if (mine && a.lse) a.lse[out] = make_float2(m, inv);
        } else {
          // among whole results, or among this block's partial ones
          float* y = it.whole ? a.full + (int64_t)(it.pre ? a.T : 0) * a.H * (D + 4)
                              : a.tile_part + (2 * (int64_t)blockIdx.x + (it.late ? 0 : 1)) * 2 * TQ * (D + 4);
          const int place = !mine ? -1 : it.whole ? (int)out : r - it.r0;
          const RowsOut<128> rows(place);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            float o[32];
            result(c, o);
            rows.write(st, reinterpret_cast<const uint4*>(o), reinterpret_cast<unsigned char*>(y + 32 * c), (D + 4) * 4);
          }
          if (mine) *reinterpret_cast<float2*>(y + (int64_t)place * (D + 4) + D) = make_float2(m, l);
          if (!it.whole && !it.late && threadIdx.x == 128)
            a.shared_items[blockIdx.x] = SharedItem{it.g.row0, it.r0, it.rows, it.h, (int)div64(it.u_last, share)};
        }
      }
      if (w == 0 || it.two) {  // the next queries may come
        umma::fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty + w);
      }
      tc_fence_before();
      if (!it.two) sides_sync();  // the second side's O has been read
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) sm100::tmem_dealloc(tmem, 512);
}

// bf16 caches (S Hk, M, D): boxes of 64 channels and TK rows of one slot's head, rows past M as zeros
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

// the queries (T, H, 2, D): boxes of 64 channels of one half, for the query heads of a key head and as many tokens as a tile has
int map_queries(CUtensorMap* m, const Args& a) {
  TmapEncodeFn fn = tmap_encode_fn();
  if (!fn) return -1;
  const cuuint32_t G = a.H / a.Hk;
  cuuint64_t dims[4] = {(cuuint64_t)a.D, 2, (cuuint64_t)a.H, (cuuint64_t)a.T};
  cuuint64_t strides[3] = {(cuuint64_t)a.D * 2, (cuuint64_t)a.D * 4, (cuuint64_t)a.H * a.D * 4};
  cuuint32_t box[4] = {64, 1, G, a.tile_rows / G}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.qw, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : -2;
}

template <int D>
int launch_dim(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, cudaStream_t st) {
  auto kernel = a.rounded ? ca_tiles<D, true> : ca_tiles<D, false>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess) return -3;
  return launch_after(kernel, a.blocks, NTHR, (int)SMEM_BYTES, st, a, mk, mv, mq) == cudaSuccess ? 0 : -4;
}

}  // namespace

int ahb::cattn::launch_tiles(const Args& a, cudaStream_t st) {
  CUtensorMap mk, mv, mq;
  if (map_cache(&mk, a.kc, a) || map_cache(&mv, a.vc, a) || map_queries(&mq, a)) return -2;
  switch (a.D) {
    case 64: return launch_dim<64>(a, mk, mv, mq, st);
    case 96: return launch_dim<96>(a, mk, mv, mq, st);
    default: return launch_dim<128>(a, mk, mv, mq, st);
  }
}
