// Attention of new tokens over a kept cache, with rows that a batch shares read once for all.
//
//   o_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = 2^(s_tj - m_t),  s_tj = sm_scale log2(e) q_t k_j
//
// over any split of the keys into ranges: each range gives (m, l = sum p, O = sum p v) and ranges join by
// m = max m_i, l = sum l_i 2^(m_i - m), O = sum O_i 2^(m_i - m).  So a prefix that a run of sequences shares is one
// range for all their rows, and a long cache is cut into ranges for as many warps as the GPU holds.
//
// Kernels: ca_append rotates the new rows and writes the cache (one more block lays the work out as units of cache
// rows); ca_tiles (cached_attention_tc.cu) takes groups of more than eight query rows, ca_rows the others; the ca_join kernels
// join what several workers or the prefix contributed; the ca_mass kernels add up what every cache row was given.
// A single token of one conversation is bound by three launches that wait for one another (13.3 us with 6 heads and 1000
// rows); batches of tokens by the cache's bytes.
#include <cfloat>
#include "cached_attention.cuh"
#include "launchers.h"
#include "mma.cuh"
#include "packed.cuh"

using namespace ahb;
using namespace ahb::cattn;

namespace {

constexpr int RW = 4, RB = 3; // warps of a block of ca_rows, its blocks on an SM (168 registers a thread)

struct Seq {
  int row0, n, slot, have, pos, pre, pre_rows;  // n = 0: padding or no token
};

// Sequence i as the arguments describe it, with everything checked that a write or read depends on.
AHB_DEVICE Seq load_seq(const Args& a, int i) {
  Seq s{0, 0, 0, 0, 0, -1, 0};
  int b, e;
  if (a.cu) {
    b = min(max(a.cu[i], 0), a.T);
    e = max(b, min(max(a.cu[i + 1], 0), a.T));
  } else {
    b = i * a.L;
    e = b + a.L;
  }
  s.row0 = b;
  s.slot = a.slots ? a.slots[i] : i;
  if ((unsigned)s.slot >= (unsigned)a.S) return s;
  s.have = a.lengths[s.slot];
  if (s.have < 0 || s.have > a.M - (e - b)) return s;
  if (a.prefix) {
    s.pre = a.prefix[i];
    if ((unsigned)s.pre < (unsigned)a.S) s.pre_rows = a.lengths[s.pre];
    if (s.pre_rows <= 0 || s.pre_rows > a.M) s.pre = -1, s.pre_rows = 0;
  }
  s.pos = a.seen ? a.seen[s.slot] : s.have + s.pre_rows;
  if (s.pos < 0 || (a.table >= 0 && s.pos > a.table - (e - b))) return s;
  s.n = e - b;
  return s;
}

// ----------------------------------------------------------------------------- new rows and the plan
constexpr int AT = 256, PT = 256;

struct Sum64 {
  AHB_DEVICE int64_t operator()(int64_t a, int64_t b) const { return a + b; }
};
struct Max64 {
  AHB_DEVICE int64_t operator()(int64_t a, int64_t b) const { return a > b ? a : b; }
};

// inclusive scan over the block's PT threads
template <class F>
AHB_DEVICE int64_t block_scan(int64_t v, int64_t* sh, F f) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = f(v, u);
  }
  __syncthreads();
  if (lane == 31) sh[w] = v;
  __syncthreads();
  for (int i = 0; i < w; ++i) v = f(v, sh[i]);
  return v;
}

// One block lays the work out: the groups, and the first unit of each in the kernel that takes it.
AHB_DEVICE void make_plan(const Args& a) {
  __shared__ int64_t sh[PT / 32];
  __shared__ int64_t carry[2 * KINDS + 1];  // sums so far, of own rows and of runs; the last run's start
  if (threadIdx.x <= 2 * KINDS) carry[threadIdx.x] = threadIdx.x == 2 * KINDS ? -1 : 0;
  for (int base = 0; base < a.B; base += PT) {
    const int i = base + (int)threadIdx.x;
    Seq s{0, 0, 0, 0, 0, -1, 0};
    int before = -1, after = -1;  // the neighbours' prefixes
    if (i < a.B) {
      s = load_seq(a, i);
      if (a.prefix && s.n > 0 && s.pre >= 0) {
        if (i > 0) {
          const Seq u = load_seq(a, i - 1);
          before = u.n > 0 ? u.pre : -1;
        }
        if (i + 1 < a.B) {
          const Seq u = load_seq(a, i + 1);
          after = u.n > 0 ? u.pre : -1;
        }
      }
    }
    const bool live = s.n > 0, starts = live && s.pre >= 0 && before != s.pre, ends = live && s.pre >= 0 && after != s.pre;
    Group own{s.row0, live ? s.n : 0, s.slot, live ? s.have + s.n : 0, s.have, 0};
    Group run{0, 0, 0, 0, 0, 0};
    if (a.prefix) {
      __syncthreads();
      const int64_t c = carry[2 * KINDS];
      const int64_t first = Max64()(c, block_scan(starts ? i : -1, sh, Max64()));
      if (ends) {
        const int row0 = a.cu ? min(max(a.cu[first], 0), a.T) : (int)first * a.L;
        run = Group{row0, s.row0 + s.n - row0, s.pre, s.pre_rows, s.pre_rows, 0};
        a.run_end[first] = i;
      }
      if (i < a.B) a.run_start[i] = live && s.pre >= 0 ? (int)first : -1;
      if (threadIdx.x == PT - 1) carry[2 * KINDS] = first;
    }
    for (int x = 0; x < (a.prefix ? 2 : 1); ++x) {
      Group& g = x ? run : own;
      int64_t units[KINDS] = {0, 0, 0};
      if (g.tokens > 0 && !is_tiles(a, g)) {
        g.per_head = row_units(g);
        units[ROWS] = a.Hk * g.per_head;
      }
      if (g.tokens > 0 && is_tiles(a, g)) {
        const int n = row_tiles(a, g);
        for (int rt = 0; rt < n; ++rt) g.per_head += tile_item(a, g, rt).units;
        units[TILES] = a.Hk * g.per_head;
      }
      if (i < a.B) a.groups[x * a.B + i] = g;
      if (a.mass && !x && g.tokens > 0) units[TILES_MASS] = is_tiles(a, g) ? (int64_t)a.Hk * ceil_div(g.keys, 4 * KU) : 0;
      for (int k = 0; k < (x || !a.mass ? 2 : KINDS); ++k) {
        __syncthreads();
        const int64_t c = carry[KINDS * x + k];
        const int64_t upto = c + block_scan(units[k], sh, Sum64());
        if (i < a.B) a.sums[k][x * (a.B + 1) + i] = upto - units[k];
        if (threadIdx.x == PT - 1) carry[KINDS * x + k] = upto;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < KINDS && (threadIdx.x < 2 || a.mass)) {
    a.sums[threadIdx.x][a.B] = carry[threadIdx.x];
    if (threadIdx.x < 2) {
      a.sums[threadIdx.x][2 * a.B + 1] = carry[KINDS + threadIdx.x];
      const int workers = threadIdx.x == TILES ? a.blocks : a.warps;
      a.shares[threadIdx.x] = workers ? share_of(carry[threadIdx.x] + carry[KINDS + threadIdx.x], workers) : 0;
    }
  }
}

// Eight channels of one half of a head and the eight of the other half that they rotate with.
template <bool VEC>
AHB_DEVICE void load8(const bf16* p, float* v) {
  if (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
  }
}
template <bool VEC>
AHB_DEVICE void load8(const float* p, float* v) {
  if (VEC) {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  }
}
// ... to p, and what their rounding leaves of them to `rest` (null: nowhere)
AHB_DEVICE void store8(bf16* p, bf16* rest, const float* v) {
  uint4 u, x;
  uint32_t *w = reinterpret_cast<uint32_t*>(&u), *y = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) split2(make_float2(sanitize(v[2 * i], CLIP), sanitize(v[2 * i + 1], CLIP)), w[i], y[i]);
  *reinterpret_cast<uint4*>(p) = u;
  if (rest) *reinterpret_cast<uint4*>(rest) = x;
}

// Block 0 makes the plan; the others rotate, clip and place `per` token rows each, and make rows of no sequence zero.
// Bound by instructions and their latency, as every pair of channels is rotated, clipped, split and rounded: 8192 tokens of 48
// heads of 128 take 52 us for 159 MB, half the copy's rate (with a thread's channels and head fixed over its rows the same).
template <bool VEC>
__global__ void __launch_bounds__(AT) ca_append(const Args a, int per) {
  next_may_start();
  if (blockIdx.x == 0) {
    make_plan(a);
    return;
  }
  __shared__ Seq s_sh;
  __shared__ int i_sh, end_sh;
  const int t_end = min(a.T, (int)blockIdx.x * per), half = a.D >> 1, pc = half >> 3, heads = a.H + 2 * a.Hk;
  for (int t = (blockIdx.x - 1) * per; t < t_end;) {
    __syncthreads();
    if (threadIdx.x == 0) {  // the rows from t on that are of one sequence, or of none
      int i = -1, end = t_end;
      if (a.cu) {  // the last sequence that starts at or before the row
        int lo = 0, hi = a.B;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (a.cu[mid] <= t) lo = mid + 1;
          else hi = mid;
        }
        i = lo - 1;
        if (lo < a.B) end = min(end, a.cu[lo]);
      } else {
        i = t / a.L;
        end = min(end, (i + 1) * a.L);
      }
      Seq s{0, 0, 0, 0, 0, -1, 0};
      if (i >= 0) s = load_seq(a, i);
      if (t < s.row0 || t >= s.row0 + s.n) i = -1;
      else end = min(end, s.row0 + s.n);
      i_sh = i;
      s_sh = s;
      end_sh = end;
    }
    __syncthreads();
    const int i = i_sh, n = end_sh - t;
    const Seq s = s_sh;
    for (int x = threadIdx.x; x < n; x += AT) a.row_seq[t + x] = i;
    if (i < 0) {
      for (int64_t x = threadIdx.x; x < (int64_t)n * a.H * a.D / 8; x += AT)
        reinterpret_cast<uint4*>(a.o + (int64_t)t * a.H * a.D)[x] = make_uint4(0, 0, 0, 0);
      t = end_sh;
      continue;
    }
    const int64_t row0 = (int64_t)s.have + t - s.row0;
    const int pos0 = s.pos + t - s.row0;
#pragma unroll 2
    for (int x = threadIdx.x; x < n * heads * pc; x += AT) {
      const int y = x / (heads * pc), z = x - y * heads * pc, h = z / pc, c = (z - h * pc) << 3;
      const int64_t row = row0 + y;
      const bf16* src;
      bf16 *dst, *rest = nullptr;
      bool turn = a.table >= 0;
      if (h < a.H) {
        src = a.q + (t + y) * a.qs + h * a.D;
        dst = a.qw + ((int64_t)(t + y) * a.H + h) * 2 * a.D;
        rest = dst + a.D;
      } else {
        const int hk = h < a.H + a.Hk ? h - a.H : h - a.H - a.Hk;
        const int64_t at = (((int64_t)s.slot * a.Hk + hk) * a.M + row) * a.D;
        if (h < a.H + a.Hk) {
          src = a.k + (t + y) * a.ks + hk * a.D;
          dst = a.kc + at;
        } else {
          src = a.v + (t + y) * a.vs + hk * a.D;
          dst = a.vc + at;
          turn = false;
        }
      }
      alignas(16) float lo[8], hi[8];
      load8<VEC>(src + c, lo);
      load8<VEC>(src + c + half, hi);
      if (turn) {
        alignas(16) float cs[8], sn[8];
        load8<VEC>(a.cos + (int64_t)(pos0 + y) * a.D + c, cs);
        load8<VEC>(a.sin + (int64_t)(pos0 + y) * a.D + c, sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x1 = lo[e], x2 = hi[e];
          lo[e] = x1 * cs[e] - x2 * sn[e];
          hi[e] = x2 * cs[e] + x1 * sn[e];
        }
      }
      if (h < a.H && a.negate) {
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = -lo[e], hi[e] = -hi[e];
      }
      store8(dst + c, rest ? rest + c : nullptr, lo);
      store8(dst + c + half, rest ? rest + c + half : nullptr, hi);
    }
    if (a.mass)
      for (int x = threadIdx.x; x < n * a.Hk; x += AT) {
        const int y = x / a.Hk, h = x - y * a.Hk;
        const int64_t at = ((int64_t)s.slot * a.Hk + h) * a.M + row0 + y;
        a.mass[at] = 0.f;
        a.held[at] = pos0 + y;
      }
    t = end_sh;
  }
}

// ----------------------------------------------------------------------------- rows against cache rows
// A unit's products on m16n8k16 tiles.  Scores: A is the queries, eight rows as rounded to bf16 and, in the
// tile's other eight rows, what the rounding left of them: the sum of the two halves is the score of the
// query in 32 bits, at no further product.  Values: A is the values' transpose, B the weights as rounded and, in a second product,
// what that left of them, so no row of the tile is idle and eight rows of O take D / 4 registers.
// Lane (g, t4) loads 16 bytes of a cache row at once: which channel a fragment's position means is free, as long as both
// operands agree.
template <int D>
AHB_DEVICE void load_q(uint32_t (&qa)[D / 16][4], const bf16* p, int t4) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint4 x = p ? *reinterpret_cast<const uint4*>(p + 32 * j + 8 * t4) : make_uint4(0, 0, 0, 0);
    const uint4 y = p ? *reinterpret_cast<const uint4*>(p + D + 32 * j + 8 * t4) : make_uint4(0, 0, 0, 0);
    qa[2 * j][0] = x.x, qa[2 * j][2] = x.y, qa[2 * j + 1][0] = x.z, qa[2 * j + 1][2] = x.w;
    qa[2 * j][1] = y.x, qa[2 * j][3] = y.y, qa[2 * j + 1][1] = y.z, qa[2 * j + 1][3] = y.w;
  }
}

// Channels 32 j + 8 t4 .. + 8 of rows g and g + 8 of the unit.
template <int D>
AHB_DEVICE void load_keys(uint4 (&kr)[2][D / 32], const bf16* base, int j0, int keys, int g, int t4) {
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      kr[x][j] = j0 + 8 * x + g < keys
                     ? *reinterpret_cast<const uint4*>(base + (int64_t)(j0 + 8 * x + g) * D + 32 * j + 8 * t4)
                     : make_uint4(0, 0, 0, 0);
}

// s[x][e]: query row g, cache row 8 x + 2 t4 + e
template <int D>
AHB_DEVICE void scores(float (&s)[2][2], const uint32_t (&qa)[D / 16][4], const uint4 (&kr)[2][D / 32]) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t b0[2] = {kr[x][j].x, kr[x][j].y}, b1[2] = {kr[x][j].z, kr[x][j].w};
      mma16816(c, qa[2 * j], b0);
      mma16816(c, qa[2 * j + 1], b1);
    }
    s[x][0] = c[0] + c[2];
    s[x][1] = c[1] + c[3];
  }
}

// Channels 64 c + 8 g .. + 8 (a last piece of 32 channels: 64 c + 4 g .. + 4) of rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9.
// Rows at or past `keys` are zero: what the cache holds there may be infinite, and 0 times that is no zero.
template <int D>
AHB_DEVICE void load_values(uint4 (&vr)[4][(D + 63) / 64], const bf16* base, int j0, int keys, int g, int t4) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int j = j0 + 2 * t4 + (x & 1) + 8 * (x >> 1);
    const bf16* p = base + (int64_t)j * D;
#pragma unroll
    for (int c = 0; c < (D + 63) / 64; ++c) {
      vr[x][c] = make_uint4(0, 0, 0, 0);
      if (j < keys) {
        if (64 * c + 64 <= D) {
          vr[x][c] = *reinterpret_cast<const uint4*>(p + 64 * c + 8 * g);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(p + 64 * c + 4 * g);
          vr[x][c].x = u.x;
          vr[x][c].y = u.y;
        }
      }
    }
  }
}

// o[4 c + j][0, 1]: channel 64 c + 8 g + 2 j (a last piece of 32: 4 g + 2 j) of query rows 2 t4 and 2 t4 + 1; [2, 3]: the next channel
template <int D>
AHB_DEVICE void add_values(float (&o)[D / 16][4], const uint32_t (&ph)[2], const uint32_t (&pl)[2],
                           const uint4 (&vr)[4][(D + 63) / 64]) {
#pragma unroll
  for (int c = 0; c < (D + 63) / 64; ++c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (64 * c + 16 * j >= D) break;
      const uint32_t w0 = (&vr[0][c].x)[j], w1 = (&vr[1][c].x)[j], w2 = (&vr[2][c].x)[j], w3 = (&vr[3][c].x)[j];
      const uint32_t va[4] = {__byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410),
                              __byte_perm(w2, w3, 0x7632)};
      mma16816(o[4 * c + j], va, ph);
      mma16816(o[4 * c + j], va, pl);
    }
  }
}

// Bound by HBM: 64 tokens over 60 to 2500 rows of 16 heads of 128, 673 MB in 111 us, 0.94 of the copy's rate; loads of the next
// unit are issued when the products have taken the last one's registers (168 a thread, 12 warps an SM).
template <int D>
__global__ void __launch_bounds__(RW * 32, RB) ca_rows(const Args a) {
  next_may_start();
  after_previous();
  constexpr int MT = D / 16, VC = (D + 63) / 64;
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int w = blockIdx.x * RW + (threadIdx.x >> 5);
  const int64_t *own = a.sums[ROWS], *runs = own + a.B + 1;
  const int64_t n_own = own[a.B], all = n_own + runs[a.B], share = share_of(all, a.warps);
  int64_t u = (int64_t)w * share;
  const int64_t u_first = u, u_end = min(u + share, all);
  const int G = a.H / a.Hk;
  while (u < u_end) {
    const bool pre = u >= n_own;
    const int i = pre ? find_group(runs, a.B, u - n_own) : find_group(own, a.B, u);
    const Group gr = a.groups[pre ? a.B + i : i];
    const int per_head = row_units(gr);
    const int64_t u0 = pre ? n_own + runs[i] : own[i];
    const int h = (int)div64(u - u0, per_head);
    const int64_t first = u0 + (int64_t)h * per_head;  // the head's units
    const int ks = (int)(u - first), ke = (int)min((int64_t)per_head, u_end - first);
    u = first + ke;
    const bf16* kb = a.kc + ((int64_t)gr.slot * a.Hk + h) * a.M * D;
    const bf16* vb = a.vc + ((int64_t)gr.slot * a.Hk + h) * a.M * D;
    uint4 kr[2][D / 32], vr[4][VC];
    load_keys<D>(kr, kb, ks * KU, gr.keys, g, t4);
    load_values<D>(vr, vb, ks * KU, gr.keys, g, t4);
    // this lane's row: row g is token g / G, query head h G + g % G
    const int tt = g / G;
    const int64_t out = g < gr.tokens * G ? (int64_t)(gr.row0 + tt) * a.H + h * G + (g - tt * G) : -1;
    const int last = min(gr.keys - 1, pre ? gr.keys : gr.before + tt);
    uint32_t qa[D / 16][4];
    load_q<D>(qa, out >= 0 ? a.qw + out * 2 * D : nullptr, t4);
    float o[MT][4], m = -INFINITY, l = 0.f;
    zero_acc<MT>(o);
    for (int c = ks; c < ke; ++c) {
      float s[2][2];
      scores<D>(s, qa, kr);
      if (c + 1 < ke) load_keys<D>(kr, kb, (c + 1) * KU, gr.keys, g, t4);
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[x][e] = c * KU + 8 * x + 2 * t4 + e <= last ? __fmul_rn(s[x][e], a.scale2) : -INFINITY;  // rounded once, for the maximum and the weights
          mx = fmaxf(mx, s[x][e]);
        }
      if (a.mass && !pre && out >= 0) {  // for ca_mass_rows
        float* y = a.scores + ((first + c) * RT + g) * KU + 2 * t4;
        *reinterpret_cast<float2*>(y) = make_float2(s[0][0], s[0][1]);
        *reinterpret_cast<float2*>(y + 8) = make_float2(s[1][0], s[1][1]);
      }
      if (__any_sync(0xffffffffu, mx > m + SLACK)) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : ex2(m - mn);
        m = mn;
        l *= f;
        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t4), f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          o[j][0] *= f0, o[j][1] *= f1;
          o[j][2] *= f0, o[j][3] *= f1;
        }
      }
      const float mr = m == -INFINITY ? 0.f : m;
      uint32_t ph[2], pl[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float2 p = make_float2(ex2(s[x][0] - mr), ex2(s[x][1] - mr));
        l += p.x + p.y;
        split2(p, ph[x], pl[x]);
      }
      add_values<D>(o, ph, pl, vr);
      if (c + 1 < ke) load_values<D>(vr, vb, (c + 1) * KU, gr.keys, g, t4);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const bool whole = ks == 0 && ke == per_head, final = whole && !a.full;
    float* part = a.part + (2 * (int64_t)w + (first >= u_first ? 1 : 0)) * RT * (D + 4);
    float* full = whole && a.full ? a.full + (int64_t)(pre ? a.T : 0) * a.H * (D + 4) : nullptr;
    const float inv = final ? 1.f / l : 1.f;
    if (t4 == 0 && out >= 0) {
      if (!final)
        *reinterpret_cast<float2*>((full ? full + out * (D + 4) : part + g * (D + 4)) + D) = make_float2(m, l);
      else if (a.lse)
        a.lse[out] = make_float2(m, inv);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // rows 2 t4 and 2 t4 + 1
      const int64_t row = __shfl_sync(0xffffffffu, out, 8 * t4 + 4 * b);
      const float f = __shfl_sync(0xffffffffu, inv, 8 * t4 + 4 * b);
      if (row < 0) continue;
      float* y = full ? full + row * (D + 4) : part + (2 * t4 + b) * (D + 4);
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const int at = 64 * c + (64 * c + 64 <= D ? 8 : 4) * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (64 * c + 16 * j >= D) break;
          const float x0 = o[4 * c + j][b], x1 = o[4 * c + j][2 + b];
          if (final) *reinterpret_cast<uint32_t*>(a.o + row * D + at + 2 * j) = pack2(x0 * f, x1 * f);
          else *reinterpret_cast<float2*>(y + at + 2 * j) = make_float2(x0, x1);
        }
      }
    }
  }
}

// ----------------------------------------------------------------------------- joining
// Partial results of one query row, a lane's channel pairs of them.
template <int D>
struct Joined {
  static constexpr int PL = (D + 63) / 64;
  float m = -INFINITY, l = 0.f;
  float2 o[PL];
  AHB_DEVICE Joined() {
#pragma unroll
    for (int c = 0; c < PL; ++c) o[c] = make_float2(0.f, 0.f);
  }
  AHB_DEVICE void one(float2 ml, const float2* v) {
    if (ml.x == -INFINITY) return;
    const float mn = fmaxf(m, ml.x), f = ex2(m - mn), e = ex2(ml.x - mn);
    m = mn;
    l = l * f + ml.y * e;
#pragma unroll
    for (int c = 0; c < PL; ++c) {
      o[c].x = o[c].x * f + v[c].x * e;
      o[c].y = o[c].y * f + v[c].y * e;
    }
  }
  // results k0 .. k1 where place(k) says, four at a time, so that their loads travel together
  template <class F>
  AHB_DEVICE void add(F place, int k0, int k1) {
    const int lane = threadIdx.x & 31;
    for (; k0 < k1; k0 += 4) {
      float2 ml[4], v[4][PL];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k0 + k >= k1) break;
        const float* p = place(k0 + k);
        ml[k] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
        for (int c = 0; c < PL; ++c)
          if (64 * c + 2 * lane < D) v[k][c] = *reinterpret_cast<const float2*>(p + 64 * c + 2 * lane);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k0 + k < k1) one(ml[k], v[k]);
    }
  }
  AHB_DEVICE void finish(const Args& a, int64_t out) const {
    const int lane = threadIdx.x & 31;
    const float inv = 1.f / l;
#pragma unroll
    for (int c = 0; c < PL; ++c)
      if (64 * c + 2 * lane < D)
        *reinterpret_cast<uint32_t*>(a.o + out * D + 64 * c + 2 * lane) = pack2(o[c].x * inv, o[c].y * inv);
    if (a.lse && lane == 0) a.lse[out] = make_float2(m, inv);
  }
};

constexpr int JW = 8;  // warps of a block

// Where the results of a token row lie: of its own rows and of its prefix's, the same for all its query heads but for `first`.
struct Source {
  bool tiles;
  int row, rows;                       // the row within a worker's partial results (of query head 0), rows of those
  int64_t base, per_head, units, share;  // key head h's first unit is base + h per_head
};
AHB_DEVICE Source source(const Args& a, const Group& g, int x, int at, int t) {
  Source s;
  s.tiles = is_tiles(a, g);
  const int64_t* own = a.sums[s.tiles ? TILES : ROWS];
  const int64_t* runs = own + a.B + 1;
  s.share = a.shares[s.tiles ? TILES : ROWS];
  s.base = x ? own[a.B] + runs[at] : own[at];
  s.row = (t - g.row0) * (a.H / a.Hk);
  s.rows = RT;
  s.per_head = g.per_head;
  s.units = s.per_head;
  if (s.tiles) {  // a token's rows are of one item
    const int rt = s.row / (2 * a.tile_rows);
    int before = 0;
    for (int k = threadIdx.x & 31; k < rt; k += 32) before += tile_item(a, g, k).units;
    s.base += __reduce_add_sync(0xffffffffu, before) + ITEM_COST;
    s.units = tile_item(a, g, rt).units - ITEM_COST;
    s.row -= rt * 2 * a.tile_rows;
    s.rows = 2 * TQ;
  }
  return s;
}

// A token row and query heads h0 .. h1, by one warp (WIDE: head h0, its partial results spread over the
// block's warps: where rows are few, every one is cut into many).  Nothing is done for what is final already.
template <int D, bool WIDE>
AHB_DEVICE void join_row(const Args& a, int t, int h0, int h1) {
  const int warp = threadIdx.x >> 5, G = a.H / a.Hk;
  const int i = a.row_seq[t];
  if (i < 0) return;
  const Group own = a.groups[i];
  if (!a.full && is_tiles(a, own)) return;  // ca_join_tiles
  const int start = a.full ? a.run_start[i] : -1, n = start >= 0 ? 2 : 1;
  Source src[2];
  src[0] = source(a, own, 0, i, t);
  if (n == 2) {
    const int end = a.run_end[start];
    src[1] = source(a, a.groups[a.B + end], 1, end, t);
  }
  for (int hq = h0; hq < h1; ++hq) {
    const int h = per_group(hq, G);
    const int64_t out = (int64_t)t * a.H + hq;
    Joined<D> sum;
    // the head's results one after another: of own rows, of the prefix's, each whole or from one worker after another
    const float* from[2] = {nullptr, nullptr};
    int64_t w0[2] = {0, 0}, slot[2] = {0, 0};
    int count[2] = {0, 0};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (x >= n) break;
      const Source& s = src[x];
      const int64_t first = s.base + h * s.per_head;
      w0[x] = div64(first, s.share);
      const int64_t rest = first + s.units - 1 - w0[x] * s.share;  // mostly one or two workers
      count[x] = rest < s.share ? 1 : rest < 2 * s.share ? 2 : 1 + (int)div64(rest, s.share);
      slot[x] = (int64_t)s.rows * (D + 4);
      from[x] = count[x] > 1 ? (s.tiles ? a.tile_part : a.part) + (int64_t)(s.row + hq - h * G) * (D + 4)
                             : a.full + ((int64_t)x * a.T * a.H + out) * (D + 4);
    }
    if (!a.full && count[0] == 1) continue;  // done
    auto place = [&](int k) {
      const bool x = k >= count[0];
      const int j = x ? k - count[0] : k;
      const int64_t at = 2 * ((x ? w0[1] : w0[0]) + j) + (j > 0 ? 0 : 1);  // the first one's second result, the others' first ones
      return (x ? from[1] : from[0]) + ((x ? count[1] : count[0]) > 1 ? at * (x ? slot[1] : slot[0]) : 0);
    };
    const int all = count[0] + count[1], each = WIDE ? (all + JW - 1) / JW : all, k0 = WIDE ? warp * each : 0;
    sum.add(place, k0, min(all, k0 + each));
    if (WIDE) {
      constexpr int PL = Joined<D>::PL;
      __shared__ float2 sh[JW][PL + 1][32];
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int c = 0; c < PL; ++c) sh[warp][c][lane] = sum.o[c];
      sh[warp][PL][lane] = make_float2(sum.m, sum.l);
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int k = 1; k < JW; ++k) {
        float2 v[PL];
#pragma unroll
        for (int c = 0; c < PL; ++c) v[c] = sh[k][c][lane];
        sum.one(sh[k][PL][lane], v);
      }
    }
    sum.finish(a, out);
  }
}
template <int D>
__global__ void __launch_bounds__(JW * 32) ca_join_wide(const Args a) {
  next_may_start();
  after_previous();
  join_row<D, true>(a, blockIdx.x, blockIdx.y, blockIdx.y + 1);
}
// A warp takes `heads` query heads of a token row: where its results lie costs more to look up than a head to join.  Bound by
// instructions, 600 a row and head: 2407 tokens of 16 heads, three or four partial results each, 39 us (one result after the other
// and all looked up by division 62).
constexpr int JB = 3;  // blocks on an SM
template <int D>
__global__ void __launch_bounds__(JW * 32, JB) ca_join(const Args a, int heads) {
  next_may_start();
  after_previous();
  if (!a.full && a.sums[ROWS][a.B] == 0) return;  // all is the tile kernel's
  const int per = (a.H + heads - 1) / heads;
  for (int64_t x = (int64_t)blockIdx.x * JW + (threadIdx.x >> 5); x < (int64_t)a.T * per; x += (int64_t)gridDim.x * JW) {
    const int t = (int)div64(x, per), h0 = (int)(x - (int64_t)t * per) * heads;
    join_row<D, false>(a, t, h0, min(a.H, h0 + heads));
  }
}

// Without a prefix only items of the tile kernel that several of its blocks share are left to join.  Block (b, y) takes
// rows 32 y .. of the item that began among block b's units and goes on behind them, as block b has noted it.
template <int D>
__global__ void __launch_bounds__(JW * 32) ca_join_tiles(const Args a) {
  next_may_start();
  after_previous();
  const SharedItem it = a.shared_items[blockIdx.x];
  const int G = a.H / a.Hk;
  const int64_t slot = 2 * TQ * (D + 4);
  for (int row = 32 * blockIdx.y + (threadIdx.x >> 5); row < min(it.rows, 32 * (int)blockIdx.y + 32); row += JW) {
    const int r = it.r0 + row, tt = per_group(r, G);
    const float* part = a.tile_part + (int64_t)row * (D + 4);
    Joined<D> sum;
    // the block's second result, then the others' first ones
    sum.add([&](int k) { return part + (2 * ((int64_t)blockIdx.x + k) + (k == 0 ? 1 : 0)) * slot; }, 0, it.last - (int)blockIdx.x + 1);
    sum.finish(a, (int64_t)(it.row0 + tt) * a.H + it.h * G + (r - tt * G));
  }
}

// ----------------------------------------------------------------------------- what every cache row was given
// Bound by latency and the scores' bytes: 48 tokens of 32 heads over 200 to 4000 rows, 14 us beside the row kernel's 73.
// Of the row kernel's groups, from the scores that it has kept (32 bytes a cache row, of its 4 D; made again from the
// keys they took as long as the row kernel itself).  A warp goes through its share of the units; lane 4 r + k has query row r
// and cache rows 4 k .. + 4.  A weight is 2^(s - m) / l, the softmax's own: with m + log2 l in one number large scores would round log2 l
// away (at scores of 1e5 a token's weights came to 1.003 or 0.997).
constexpr int MB = 12;  // blocks of ca_mass_rows on an SM
__global__ void __launch_bounds__(RW * 32, MB) ca_mass_rows(const Args a, int warps) {
  next_may_start();
  after_previous();
  const int lane = threadIdx.x & 31, G = a.H / a.Hk, r = lane >> 2, tt = per_group(r, G), k0 = 4 * (lane & 3);
  const int64_t* units = a.sums[ROWS];
  const int64_t all = units[a.B], share = share_of(all, warps);
  int64_t u = ((int64_t)blockIdx.x * RW + (threadIdx.x >> 5)) * share;
  const int64_t u_end = min(u + share, all);
  while (u < u_end) {
    const int i = find_group(units, a.B, u);
    const Group gr = a.groups[i];
    const int per_head = row_units(gr), h = (int)div64(u - units[i], per_head), c0 = (int)(u - units[i] - (int64_t)h * per_head);
    const int n = (int)min((int64_t)(per_head - c0), u_end - u);
    const bool in = r < gr.tokens * G;
    const float2 ml = in ? a.lse[(int64_t)(gr.row0 + tt) * a.H + h * G + r - tt * G] : make_float2(0.f, 0.f);
    float* m = a.mass + ((int64_t)gr.slot * a.Hk + h) * a.M;
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      float4 p = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in) {
        const float4 s = *reinterpret_cast<const float4*>(a.scores + (u + c) * RT * KU + lane * 4);
        p = make_float4(ex2(s.x - ml.x) * ml.y, ex2(s.y - ml.x) * ml.y, ex2(s.z - ml.x) * ml.y, ex2(s.w - ml.x) * ml.y);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        p.x += __shfl_xor_sync(0xffffffffu, p.x, o);
        p.y += __shfl_xor_sync(0xffffffffu, p.y, o);
        p.z += __shfl_xor_sync(0xffffffffu, p.z, o);
        p.w += __shfl_xor_sync(0xffffffffu, p.w, o);
      }
      const int x = lane >> 2, j = (c0 + c) * KU + k0 + x;  // lanes 0 .. 15: a cache row each
      const float mine = x == 0 ? p.x : x == 1 ? p.y : x == 2 ? p.z : p.w;
      if (x < 4 && j < gr.keys) m[j] += mine;
    }
    u += n;
  }
}

// Of the tile kernel's: a warp holds 64 cache rows and goes over the query rows that see them, eight at a time:
// sum_t 2^(s_tj - m_t) / l_t.  The scores are summed in another order than the tile kernel's, which moves a weight by some 2^-22 of its
// row's largest score: next to nothing at scores of tens, 2 % at 1e5; more than the query rows that see a cache row it never gathers.  Bound by the products, each query tile with its rounding remainders: a tracked prompt of 4000 tokens
// takes 694 us in all, 172 untracked (16 cache rows a warp: 1017).
constexpr int KM = 4;  // units of 16 cache rows that a warp holds
template <int D, bool ROUNDED>
__global__ void __launch_bounds__(RW * 32, 2) ca_mass(const Args a) {
  next_may_start();
  after_previous();
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int64_t* units = a.sums[TILES_MASS];
  const int64_t all = units[a.B];
  const int G = a.H / a.Hk;
  for (int64_t u = (int64_t)blockIdx.x * RW + (threadIdx.x >> 5); u < all; u += (int64_t)gridDim.x * RW) {
    const int i = find_group(units, a.B, u);
    const Group gr = a.groups[i];
    const int per_head = ceil_div(gr.keys, KM * KU), h = (int)div64(u - units[i], per_head);
    const int j0 = (int)(u - units[i] - (int64_t)h * per_head) * KM * KU;
    uint4 kr[KM][2][D / 32];
#pragma unroll
    for (int y = 0; y < KM; ++y) load_keys<D>(kr[y], a.kc + ((int64_t)gr.slot * a.Hk + h) * a.M * D, j0 + y * KU, gr.keys, g, t4);
    float sum[KM][2][2] = {};
    const int rows = gr.tokens * G;
    // from the first token that sees row j0
    for (int r0 = max(0, j0 - gr.before) * G / RT * RT; r0 < rows; r0 += RT) {
      const int r = r0 + g, tt = per_group(r, G);
      const int64_t out = (int64_t)(gr.row0 + tt) * a.H + h * G + (r - tt * G);
      const float2 ml = r < rows ? a.lse[out] : make_float2(0.f, 0.f);
      const int last = r < rows ? gr.before + tt : -1;
      uint32_t qa[D / 16][4];
      load_q<D>(qa, r < rows ? a.qw + out * 2 * D : nullptr, t4);
#pragma unroll
      for (int y = 0; y < KM; ++y) {
        float s[2][2];
        scores<D>(s, qa, kr[y]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (j0 + y * KU + 8 * x + 2 * t4 + e <= last) sum[y][x][e] += ex2(ROUNDED ? __fadd_rn(__fmul_rn(s[x][e], a.scale2), -ml.x) : __fmaf_rn(s[x][e], a.scale2, -ml.x)) * ml.y;
      }
    }
#pragma unroll
    for (int y = 0; y < KM; ++y)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = sum[y][x][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          const int j = j0 + y * KU + 8 * x + 2 * t4 + e;
          if (g == 0 && j < gr.keys) a.mass[((int64_t)gr.slot * a.Hk + h) * a.M + j] += fminf(v, (float)rows);
        }
  }
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Places the workspace's parts (base null: only counts) and returns its bytes.
int64_t lay_out(Args& a, char* base) {
  int64_t at = 0;
  auto place = [&](int64_t bytes) {
    char* p = base ? base + at : nullptr;
    at += align256(bytes);
    return p;
  };
  const int64_t rows = (int64_t)a.T * a.H;
  const int sms = sm_count(), G = a.H / a.Hk;
  a.tile_rows = TQ / G * G;
  a.warps = sms * RB * RW;
  // no group takes tiles if there is no run and every sequence has few rows
  a.blocks = a.prefix || a.cu || a.L * G > RT ? sms : 0;
  a.qw = (bf16*)place(rows * a.D * 4);
  a.row_seq = (int*)place((int64_t)a.T * 4);
  a.groups = (Group*)place((int64_t)2 * a.B * sizeof(Group));
  a.run_start = (int*)place((int64_t)a.B * 4);
  a.run_end = (int*)place((int64_t)a.B * 4);
  for (int k = 0; k < (a.mass ? KINDS : 2); ++k) a.sums[k] = (int64_t*)place((int64_t)2 * (a.B + 1) * 8);
  a.scores = a.mass ? (float*)place((int64_t)a.B * a.Hk * ((a.M + KU - 1) / KU) * RT * KU * 4) : nullptr;
  a.lse = a.mass ? (float2*)place(rows * 8) : nullptr;
  a.part = (float*)place((int64_t)2 * a.warps * RT * (a.D + 4) * 4);
  a.tile_part = (float*)place((int64_t)2 * a.blocks * 2 * TQ * (a.D + 4) * 4);
  a.shares = (int64_t*)place(2 * 8);
  a.shared_items = (SharedItem*)place((int64_t)a.blocks * sizeof(SharedItem));
  a.full = a.prefix ? (float*)place(2 * rows * (a.D + 4) * 4) : nullptr;
  return at;
}

template <int D>
int launch(const Args& a, cudaStream_t st) {
  if (a.blocks) {
    const int rc = launch_tiles(a, st);
    if (rc) return rc;
  }
  cudaError_t e = cudaSuccess;
  // behind the tile kernel not before it has ended: its waiting blocks would sit on the SMs that the first of them leave
  // (one token of 64 conversations on a prefix 99 us, so 88)
  if (a.blocks) ca_rows<D><<<a.warps / RW, RW * 32, 0, st>>>(a);
  else e = launch_after(ca_rows<D>, a.warps / RW, RW * 32, 0, st, a);
  const int sms = a.warps / (RB * RW);
  // as many heads a warp as make four rounds of warps
  const int64_t each = ((int64_t)a.T * a.H + 4 * sms * JB * JW - 1) / (4 * sms * JB * JW);
  const int heads = each < a.H ? (int)each : a.H;
  const int64_t blocks = ((int64_t)a.T * ((a.H + heads - 1) / heads) + JW - 1) / JW;
  auto then = [&](cudaError_t next) { e = e == cudaSuccess ? next : e; };
  if (a.blocks && !a.full) then(launch_after(ca_join_tiles<D>, dim3(a.blocks, 2 * TQ / 32), JW * 32, 0, st, a));
  if ((int64_t)a.T * a.H <= 4 * sms) then(launch_after(ca_join_wide<D>, dim3(a.T, a.H), JW * 32, 0, st, a));
  else then(launch_after(ca_join<D>, (unsigned)(blocks < 16 * sms ? blocks : 16 * sms), JW * 32, 0, st, a, heads));
  if (a.mass) {
    then(launch_after(ca_mass_rows, sms * MB, RW * 32, 0, st, a, sms * MB * RW));
    if (a.blocks) then(launch_after(a.rounded ? ca_mass<D, true> : ca_mass<D, false>, sms * 2, RW * 32, 0, st, a));
  }
  if (e != cudaSuccess) return -4;
  return 0;
}

}  // namespace

int64_t ahb_cached_attention_bytes(const Args& args) {
  Args a = args;
  return lay_out(a, nullptr);
}

int ahb_cached_attention(const Args& args, void* work, cudaStream_t st) {
  Args a = args;
  a.negate = a.scale2 < 0.f;  // the queries take the scale's sign: the largest product is then the largest score
  // A masked score is -inf before it is scaled, and -inf times 0 is none: the least normal number gives the same weights
  a.scale2 = fmaxf(a.scale2 < 0.f ? -a.scale2 : a.scale2, FLT_MIN);
  a.rounded = a.scale2 * a.D * CLIP * CLIP > 268435456.f;  // queries and keys are clipped to CLIP
  lay_out(a, (char*)work);
  const bool vec = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.cos | (uintptr_t)a.sin) & 15) == 0 && ((a.qs | a.ks | a.vs) & 7) == 0;
  const int per = 1 + (a.T - 1) / (8 * sm_count()), blocks = 1 + (a.T + per - 1) / per;  // eight blocks an SM at most
  if (vec) ca_append<true><<<blocks, AT, 0, st>>>(a, per);
  else ca_append<false><<<blocks, AT, 0, st>>>(a, per);
  switch (a.D) {
    case 64: return launch<64>(a, st);
    case 96: return launch<96>(a, st);
    case 128: return launch<128>(a, st);
    default: return -1;
  }
}
