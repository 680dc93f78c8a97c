// Attention of new tokens over a kept cache, with rows that a batch shares read once for all.
//
//   o_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = 2^(s_tj - m_t),  s_tj = sm_scale log2(e) q_t k_j
//
// over any split of the keys into ranges: each range gives (m, l = sum p, O = sum p v) and ranges join by
// m = max m_i, l = sum l_i 2^(m_i - m), O = sum O_i 2^(m_i - m).  So a prefix that a run of sequences shares is one
// range for all their rows, and a long cache is cut into ranges for as many warps as the GPU holds.
//
// Kernels: ca_append rotates the new rows and writes the cache (one block a token row; one more block lays the
// work out as units of 16 cache rows); ca_rows gives every warp the same number of units, one after another;
// ca_join joins what several warps or the prefix contributed; ca_mass adds up what every cache row was given.
#include "cached_attention.h"
#include "common.cuh"
#include "launchers.h"
#include "mma.cuh"
#include "packed.cuh"

using namespace ahb;
using namespace ahb::cattn;

namespace {

constexpr int KU = 16;        // cache rows of a unit
constexpr int RT = 16;        // query rows of an item
constexpr int RW = 4;         // warps of a block of ca_rows
constexpr float CLIP = 1e3f;
constexpr float SLACK = 8.f;  // the running maximum moves when a score passes it by more than 2^8: p <= 256, and no sum nears overflow

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

AHB_DEVICE int ceil_div(int a, int b) { return (a + b - 1) / b; }
AHB_DEVICE int row_tiles(const Args& a, int tokens) { return ceil_div(tokens * (a.H / a.Hk), RT); }
AHB_DEVICE int64_t group_units(const Args& a, const Group& g) {
  return (int64_t)a.Hk * row_tiles(a, g.tokens) * ceil_div(g.keys, KU);
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

AHB_DEVICE void make_plan(const Args& a) {
  __shared__ int64_t sh[4][PT / 32];
  __shared__ int64_t carry[4];
  if (threadIdx.x < 4) carry[threadIdx.x] = threadIdx.x == 3 ? -1 : 0;
  int64_t *own = a.units, *runs = own + a.B + 1, *mass = runs + a.B + 1;
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
    const bool live = s.n > 0;
    const bool starts = live && s.pre >= 0 && before != s.pre, ends = live && s.pre >= 0 && after != s.pre;
    const Group g{s.row0, live ? s.n : 0, s.slot, live ? s.have + s.n : 0, s.have};
    const int64_t u_own = group_units(a, g), u_mass = a.mass ? (int64_t)a.Hk * ceil_div(g.keys, KU) : 0;
    __syncthreads();
    const int64_t c_own = carry[0], c_runs = carry[1], c_mass = carry[2], c_start = carry[3];
    const int64_t i_own = c_own + block_scan(u_own, sh[0], Sum64());
    const int64_t i_mass = c_mass + block_scan(u_mass, sh[1], Sum64());
    const int64_t first = Max64()(c_start, block_scan(starts ? i : -1, sh[2], Max64()));
    Group r{0, 0, 0, 0, 0};
    if (ends) {
      const int row0 = a.cu ? min(max(a.cu[first], 0), a.T) : (int)first * a.L;
      r = Group{row0, s.row0 + s.n - row0, s.pre, s.pre_rows, s.pre_rows};
      a.run_end[first] = i;
    }
    const int64_t u_runs = group_units(a, r);
    const int64_t i_runs = c_runs + block_scan(u_runs, sh[3], Sum64());
    if (i < a.B) {
      a.groups[i] = g;
      a.groups[a.B + i] = r;
      own[i] = i_own - u_own;
      runs[i] = i_runs - u_runs;
      mass[i] = i_mass - u_mass;
      a.run_start[i] = live && s.pre >= 0 ? (int)first : -1;
    }
    if (threadIdx.x == PT - 1) {
      carry[0] = i_own;
      carry[1] = i_runs;
      carry[2] = i_mass;
      carry[3] = first;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    own[a.B] = carry[0];
    runs[a.B] = carry[1];
    mass[a.B] = carry[2];
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
AHB_DEVICE void store8(bf16* p, const float* v) {
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(sanitize(v[2 * i], CLIP), sanitize(v[2 * i + 1], CLIP));
  *reinterpret_cast<uint4*>(p) = u;
}

// Block 0 makes the plan; every other block rotates, clips and places one token row.
template <bool VEC>
__global__ void __launch_bounds__(AT) ca_append(const Args a) {
  if (blockIdx.x == 0) {
    make_plan(a);
    return;
  }
  __shared__ Seq s_sh;
  __shared__ int i_sh;
  const int t = blockIdx.x - 1;
  if (threadIdx.x == 0) {
    int i = -1;
    if (a.cu) {  // the last sequence that starts at or before the row
      int lo = 0, hi = a.B;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid + 1;
        else hi = mid;
      }
      i = lo - 1;
    } else {
      i = t / a.L;
    }
    Seq s{0, 0, 0, 0, 0, -1, 0};
    if (i >= 0) s = load_seq(a, i);
    if (t < s.row0 || t >= s.row0 + s.n) i = -1;
    a.row_seq[t] = i;
    i_sh = i;
    s_sh = s;
  }
  __syncthreads();
  if (i_sh < 0) return;
  const Seq s = s_sh;
  const int tt = t - s.row0, half = a.D >> 1, per = half >> 3;
  const int64_t row = (int64_t)s.have + tt;
  const float* cs = a.table >= 0 ? a.cos + (int64_t)(s.pos + tt) * a.D : nullptr;
  const float* sn = a.table >= 0 ? a.sin + (int64_t)(s.pos + tt) * a.D : nullptr;
  const int heads = a.H + 2 * a.Hk;
  for (int x = threadIdx.x; x < heads * per; x += AT) {
    const int h = x / per, c = (x - h * per) << 3;
    const bf16* src;
    bf16* dst;
    bool turn = cs != nullptr;
    if (h < a.H) {
      src = a.q + (int64_t)t * a.qs + h * a.D;
      dst = a.qw + ((int64_t)t * a.H + h) * a.D;
    } else {
      const int hk = h < a.H + a.Hk ? h - a.H : h - a.H - a.Hk;
      const int64_t at = (((int64_t)s.slot * a.Hk + hk) * a.M + row) * a.D;
      if (h < a.H + a.Hk) {
        src = a.k + (int64_t)t * a.ks + hk * a.D;
        dst = a.kc + at;
      } else {
        src = a.v + (int64_t)t * a.vs + hk * a.D;
        dst = a.vc + at;
        turn = false;
      }
    }
    float lo[8], hi[8];
    load8<VEC>(src + c, lo);
    load8<VEC>(src + c + half, hi);
    if (turn) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x1 = lo[i], x2 = hi[i];
        lo[i] = x1 * cs[c + i] - x2 * sn[c + i];
        hi[i] = x2 * cs[c + half + i] + x1 * sn[c + half + i];
      }
    }
    store8(dst + c, lo);
    store8(dst + c + half, hi);
  }
  if (a.mass)
    for (int h = threadIdx.x; h < a.Hk; h += AT) {
      const int64_t at = ((int64_t)s.slot * a.Hk + h) * a.M + row;
      a.mass[at] = 0.f;
      a.held[at] = s.pos + tt;
    }
}

// ----------------------------------------------------------------------------- rows against cache rows
// The group whose units hold unit u: the last i with sums[i] <= u (one probe a lane, 32 ways a step).
AHB_DEVICE int find_group(const int64_t* sums, int n, int64_t u) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // sums[lo] <= u < sums[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int at = lo + (lane + 1) * step;
    const bool in = at < hi && sums[at] <= u;
    const int k = __popc(__ballot_sync(0xffffffffu, in));
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Units a warp: equal shares of all units.
AHB_DEVICE int64_t warp_share(int64_t units, int warps) { return (units + warps - 1) / warps; }

// Channels of a lane in 32-channel (scores) and 64-channel (values) pieces of a head.  A lane loads 16
// bytes of a cache row at once; which channel a fragment's position means is free, as long as both operands agree.
template <int D>
struct Frag {
  static constexpr int KJ = D / 32;            // 32-channel pieces: two k steps each
  static constexpr int VC = (D + 63) / 64;     // 64-channel pieces; the last one of 96 channels has 32
  static constexpr int NT = D / 8;             // n tiles of O
};

template <int D>
AHB_DEVICE void load_q(uint32_t (&qa)[D / 16][4], const bf16* g0, const bf16* g1, int t4) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint4 x = g0 ? *reinterpret_cast<const uint4*>(g0 + 32 * j + 8 * t4) : make_uint4(0, 0, 0, 0);
    const uint4 y = g1 ? *reinterpret_cast<const uint4*>(g1 + 32 * j + 8 * t4) : make_uint4(0, 0, 0, 0);
    qa[2 * j][0] = x.x, qa[2 * j][2] = x.y, qa[2 * j + 1][0] = x.z, qa[2 * j + 1][2] = x.w;
    qa[2 * j][1] = y.x, qa[2 * j][3] = y.y, qa[2 * j + 1][1] = y.z, qa[2 * j + 1][3] = y.w;
  }
}

// The 16 rows of a unit as operands of the scores: lane (g, t4) holds channels 32 j + 8 t4 .. + 8 of rows g and g + 8.
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

template <int D>
AHB_DEVICE void scores(float (&s)[2][4], const uint32_t (&qa)[D / 16][4], const uint4 (&kr)[2][D / 32]) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t b0[2] = {kr[x][j].x, kr[x][j].y}, b1[2] = {kr[x][j].z, kr[x][j].w};
      mma16816(s[x], qa[2 * j], b0);
      mma16816(s[x], qa[2 * j + 1], b1);
    }
  }
}

// The same rows as operands of p v: lane (g, t4) holds channels 64 c + 8 g .. + 8 (a last piece of 32
// channels: 64 c + 4 g .. + 4) of rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9.  Rows at or past `keys` are zero: what the
// cache holds there may be infinite, and 0 times that is no zero.
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

// channel e (0 .. 7) of rows a and b as one operand register
AHB_DEVICE uint32_t pair(const uint4& a, const uint4& b, int e) {
  const uint32_t x = (&a.x)[e >> 1], y = (&b.x)[e >> 1];
  return (e & 1) ? __byte_perm(x, y, 0x7632) : __byte_perm(x, y, 0x5410);
}

template <int D>
AHB_DEVICE void add_values(float (&o)[D / 8][4], const uint32_t (&pa)[4], const uint4 (&vr)[4][(D + 63) / 64]) {
#pragma unroll
  for (int c = 0; c < (D + 63) / 64; ++c) {
    const int nt = 64 * c + 64 <= D ? 8 : 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= nt) break;
      const uint32_t b[2] = {pair(vr[0][c], vr[1][c], e), pair(vr[2][c], vr[3][c], e)};
      mma16816(o[8 * c + e], pa, b);
    }
  }
}

// First channel of the run of channels that n tiles 8 c .. hold in a lane, in order: column 2 t4 of tiles e = 0, 1, ..
// and then column 2 t4 + 1 of them.
AHB_DEVICE int lane_channel(int c, int t4, int width) { return 64 * c + 2 * width * t4; }

template <int D>
__global__ void __launch_bounds__(RW * 32) ca_rows(const Args a) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int w = blockIdx.x * RW + (threadIdx.x >> 5);
  const int64_t *own = a.units, *runs = own + a.B + 1;
  const int64_t n_own = own[a.B], all = n_own + runs[a.B], share = warp_share(all, a.warps);
  int64_t u = (int64_t)w * share;
  const int64_t u_first = u, u_end = min(u + share, all);
  const int G = a.H / a.Hk;
  while (u < u_end) {
    const bool pre = u >= n_own;
    const int i = pre ? find_group(runs, a.B, u - n_own) : find_group(own, a.B, u);
    const Group gr = a.groups[pre ? a.B + i : i];
    const int per_item = ceil_div(gr.keys, KU), tiles = row_tiles(a, gr.tokens);
    const int64_t u0 = pre ? n_own + runs[i] : own[i];
    const int64_t item = (u - u0) / per_item;
    const int64_t first = u0 + item * per_item;       // the item's units
    const int ks = (int)(u - first), ke = (int)min((int64_t)per_item, u_end - first);
    const int h = (int)(item / tiles), r0 = (int)(item - (int64_t)h * tiles) * RT;
    u = first + ke;
    const bf16* kb = a.kc + ((int64_t)gr.slot * a.Hk + h) * a.M * D;
    const bf16* vb = a.vc + ((int64_t)gr.slot * a.Hk + h) * a.M * D;
    // rows of this lane: g and g + 8 of the tile; row r is token r / G, query head h G + r % G
    const int rows = gr.tokens * G;
    const bf16* qp[2];
    int64_t out[2];
    int last[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = r0 + g + 8 * x, tt = r / G;
      out[x] = r < rows ? (int64_t)(gr.row0 + tt) * a.H + h * G + (r - tt * G) : -1;
      qp[x] = out[x] >= 0 ? a.qw + out[x] * D : nullptr;
      last[x] = min(gr.keys - 1, pre ? gr.keys : gr.before + tt);
    }
    uint32_t qa[D / 16][4];
    load_q<D>(qa, qp[0], qp[1], t4);
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    zero_acc<D / 8>(o);
    uint4 kr[2][D / 32], vr[4][(D + 63) / 64];
    load_keys<D>(kr, kb, ks * KU, gr.keys, g, t4);
    load_values<D>(vr, vb, ks * KU, gr.keys, g, t4);
    for (int c = ks; c < ke; ++c) {
      float s[2][4];
      scores<D>(s, qa, kr);
      if (c + 1 < ke) load_keys<D>(kr, kb, (c + 1) * KU, gr.keys, g, t4);
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = c * KU + 8 * x + 2 * t4 + (e & 1);
          s[x][e] = j <= last[e >> 1] ? s[x][e] * a.scale2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[x][e]);
        }
      if (__any_sync(0xffffffffu, mx[0] > m[0] + SLACK || mx[1] > m[1] + SLACK)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
          mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
          const float mn = fmaxf(m[x], mx[x]);
          const float f = m[x] == -INFINITY ? 0.f : ex2(m[x] - mn);
          m[x] = mn;
          l[x] *= f;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[j][2 * x] *= f;
            o[j][2 * x + 1] *= f;
          }
        }
      }
      // p rounded to bf16 for its product with the values (relative 2^-9 each, averaging out); l sums what was not rounded
      uint32_t pa[4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mr = m[r] == -INFINITY ? 0.f : m[r];
          const float p0 = ex2(s[x][2 * r] - mr), p1 = ex2(s[x][2 * r + 1] - mr);
          l[r] += p0 + p1;
          pa[2 * x + r] = pack2(p0, p1);
        }
      add_values<D>(o, pa, vr);
      if (c + 1 < ke) load_values<D>(vr, vb, (c + 1) * KU, gr.keys, g, t4);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    const bool whole = ks == 0 && ke == per_item;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (out[x] < 0) continue;
      if (whole && !a.full) {  // final
        const float inv = 1.f / l[x];
        bf16* y = a.o + out[x] * D;
#pragma unroll
        for (int c = 0; c < (D + 63) / 64; ++c) {
          const int nt = 64 * c + 64 <= D ? 8 : 4;
          bf16* p = y + lane_channel(c, t4, nt);
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
              if (e < nt)
                *reinterpret_cast<uint32_t*>(p + b * nt + e) =
                    pack2(o[8 * c + e][2 * x + b] * inv, o[8 * c + e + 1][2 * x + b] * inv);
        }
        if (a.lse && t4 == 0) a.lse[out[x]] = m[x] + log2f(l[x]);
      } else {
        float* y = whole ? a.full + ((int64_t)(pre ? a.T : 0) * a.H + out[x]) * (D + 2)
                         : a.part + ((2 * (int64_t)w + (first >= u_first ? 1 : 0)) * RT + g + 8 * x) * (D + 2);
#pragma unroll
        for (int c = 0; c < (D + 63) / 64; ++c) {
          const int nt = 64 * c + 64 <= D ? 8 : 4;
          float* p = y + lane_channel(c, t4, nt);
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
              if (e < nt)
                *reinterpret_cast<float2*>(p + b * nt + e) =
                    make_float2(o[8 * c + e][2 * x + b], o[8 * c + e + 1][2 * x + b]);
        }
        if (t4 == 0) *reinterpret_cast<float2*>(y + D) = make_float2(m[x], l[x]);
      }
    }
  }
}

// ----------------------------------------------------------------------------- joining
// One warp for each row and query head.  Zeros for rows of no sequence; nothing for what ca_rows has finished.
template <int D>
__global__ void __launch_bounds__(128) ca_join(const Args a) {
  constexpr int PL = (D + 63) / 64;  // channel pairs of a lane
  const int lane = threadIdx.x & 31;
  const int64_t out = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (out >= (int64_t)a.T * a.H) return;
  const int t = (int)(out / a.H), hq = (int)(out - (int64_t)t * a.H), G = a.H / a.Hk, h = hq / G;
  const int i = a.row_seq[t];
  if (i < 0) {
#pragma unroll
    for (int c = 0; c < PL; ++c)
      if (64 * c + 2 * lane < D) *reinterpret_cast<uint32_t*>(a.o + out * D + 64 * c + 2 * lane) = 0u;
    return;
  }
  const int64_t *own = a.units, *runs = own + a.B + 1;
  const int64_t n_own = own[a.B], share = warp_share(n_own + runs[a.B], a.warps);
  float m = -INFINITY, l = 0.f;
  float2 o[PL];
#pragma unroll
  for (int c = 0; c < PL; ++c) o[c] = make_float2(0.f, 0.f);
  auto add = [&](const float* y) {
    const float2 ml = *reinterpret_cast<const float2*>(y + D);
    const float mn = fmaxf(m, ml.x);
    const float f = m == -INFINITY ? 0.f : ex2(m - mn), e = ml.x == -INFINITY ? 0.f : ex2(ml.x - mn);
    m = mn;
    l = l * f + ml.y * e;
#pragma unroll
    for (int c = 0; c < PL; ++c)
      if (64 * c + 2 * lane < D) {
        const float2 v = *reinterpret_cast<const float2*>(y + 64 * c + 2 * lane);
        o[c].x = o[c].x * f + v.x * e;
        o[c].y = o[c].y * f + v.y * e;
      }
  };
  for (int src = 0; src < (a.full ? 2 : 1); ++src) {
    int j = i;
    if (src == 1) {  // the run that this sequence is in
      const int start = a.run_start[i];
      if (start < 0) break;
      j = a.run_end[start];
    }
    const Group gr = a.groups[src * a.B + j];
    const int r = (t - gr.row0) * G + hq - h * G, per_item = ceil_div(gr.keys, KU);
    const int64_t first =
        (src ? n_own + runs[j] : own[j]) + ((int64_t)h * row_tiles(a, gr.tokens) + r / RT) * per_item;
    const int64_t w0 = first / share, w1 = (first + per_item - 1) / share;
    if (w0 == w1) {
      if (!a.full) return;  // final already
      add(a.full + ((int64_t)src * a.T * a.H + out) * (D + 2));
    } else {
      for (int64_t w = w0; w <= w1; ++w)
        add(a.part + ((2 * w + (first >= w * share ? 1 : 0)) * RT + r % RT) * (D + 2));
    }
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int c = 0; c < PL; ++c)
    if (64 * c + 2 * lane < D)
      *reinterpret_cast<uint32_t*>(a.o + out * D + 64 * c + 2 * lane) = pack2(o[c].x * inv, o[c].y * inv);
  if (a.lse && lane == 0) a.lse[out] = m + log2f(l);
}

// ----------------------------------------------------------------------------- what every cache row was given
// A warp holds 16 cache rows and goes over the query rows that see them: sum_t 2^(s_tj - lse_t).
template <int D>
__global__ void __launch_bounds__(RW * 32) ca_mass(const Args a) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int64_t* units = a.units + 2 * (a.B + 1);
  const int64_t all = units[a.B];
  const int G = a.H / a.Hk;
  for (int64_t u = (int64_t)blockIdx.x * RW + (threadIdx.x >> 5); u < all; u += (int64_t)gridDim.x * RW) {
    const int i = find_group(units, a.B, u);
    const Group gr = a.groups[i];
    const int per_head = ceil_div(gr.keys, KU), h = (int)((u - units[i]) / per_head);
    const int j0 = (int)(u - units[i] - (int64_t)h * per_head) * KU;
    uint4 kr[2][D / 32];
    load_keys<D>(kr, a.kc + ((int64_t)gr.slot * a.Hk + h) * a.M * D, j0, gr.keys, g, t4);
    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    const int rows = gr.tokens * G;
    // the first token that sees row j0
    for (int r0 = max(0, j0 - gr.before) * G / RT * RT; r0 < rows; r0 += RT) {
      const bf16* qp[2];
      float lse[2];
      int last[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + g + 8 * x, tt = r / G;
        const int64_t out = (int64_t)(gr.row0 + tt) * a.H + h * G + (r - tt * G);
        qp[x] = r < rows ? a.qw + out * D : nullptr;
        lse[x] = r < rows ? a.lse[out] : 0.f;
        last[x] = r < rows ? gr.before + tt : -1;
      }
      uint32_t qa[D / 16][4];
      load_q<D>(qa, qp[0], qp[1], t4);
      float s[2][4];
      scores<D>(s, qa, kr);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 8 * x + 2 * t4 + (e & 1);
          if (j <= last[e >> 1]) sum[x][e & 1] += ex2(s[x][e] * a.scale2 - lse[e >> 1]);
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[x][e] += __shfl_xor_sync(0xffffffffu, sum[x][e], o);
        const int j = j0 + 8 * x + 2 * t4 + e;
        if (g == 0 && j < gr.keys) a.mass[((int64_t)gr.slot * a.Hk + h) * a.M + j] += sum[x][e];
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
  a.warps = sm_count() * 4 * RW;
  a.qw = (bf16*)place(rows * a.D * 2);
  a.row_seq = (int*)place((int64_t)a.T * 4);
  a.groups = (Group*)place((int64_t)2 * a.B * sizeof(Group));
  a.run_start = (int*)place((int64_t)a.B * 4);
  a.run_end = (int*)place((int64_t)a.B * 4);
  a.units = (int64_t*)place((int64_t)3 * (a.B + 1) * 8);
  a.lse = a.mass ? (float*)place(rows * 4) : nullptr;
  a.part = (float*)place((int64_t)2 * a.warps * RT * (a.D + 2) * 4);
  a.full = a.prefix ? (float*)place(2 * rows * (a.D + 2) * 4) : nullptr;
  return at;
}

template <int D>
void launch(const Args& a, cudaStream_t st) {
  ca_rows<D><<<a.warps / RW, RW * 32, 0, st>>>(a);
  ca_join<D><<<(unsigned)(((int64_t)a.T * a.H + 3) / 4), 128, 0, st>>>(a);
  if (a.mass) ca_mass<D><<<a.warps / RW, RW * 32, 0, st>>>(a);
}

}  // namespace

int64_t ahb_cached_attention_bytes(const ahb::cattn::Args& args) {
  Args a = args;
  return lay_out(a, nullptr);
}

int ahb_cached_attention(const ahb::cattn::Args& args, void* work, cudaStream_t st) {
  Args a = args;
  lay_out(a, (char*)work);
  const bool vec = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 && ((a.qs | a.ks | a.vs) & 7) == 0;
  if (vec) ca_append<true><<<a.T + 1, AT, 0, st>>>(a);
  else ca_append<false><<<a.T + 1, AT, 0, st>>>(a);
  switch (a.D) {
    case 64: launch<64>(a, st); break;
    case 96: launch<96>(a, st); break;
    case 128: launch<128>(a, st); break;
    default: return -1;
  }
  return 0;
}
