// Device code that the kernels of cached attention share: how work is numbered and found.
#pragma once
#include "cached_attention.h"
#include "common.cuh"

namespace ahb {
namespace cattn {

// The kernels of a call follow one another closely: each lets the next one start while it runs (its blocks take the places
// that become free), and waits for the one before, whole and with all that it wrote, before it reads anything.
AHB_DEVICE void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
AHB_DEVICE void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... A>
inline cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int block, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

constexpr int KU = 16;    // row kernel: cache rows of a unit
constexpr int RT = 8;     // ... and the query rows that it takes
constexpr int TK = 64;    // tile kernel: cache rows of a block
constexpr int TQ = 128;   // ... rows of a tensor-core tile, a.tile_rows of them used; an item has one or two tiles
constexpr float CLIP = 1e3f;
constexpr float SLACK = 8.f;  // the running maximum moves when a score passes it by more than 2^8: p <= 256, and no sum nears overflow
AHB_DEVICE int ceil_div(int a, int b) { return (a + b - 1) / b; }
// a / b of non-negative numbers that are seldom past 32 bits
AHB_DEVICE int64_t div64(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// r / G, G mostly 1
AHB_DEVICE int per_group(int r, int G) { return G == 1 ? r : r / G; }
AHB_DEVICE int query_rows(const Args& a, const Group& g) { return g.tokens * (a.H / a.Hk); }

// Which kernel takes a group: up to eight query rows leave a 128-row tile idle and need no tile to be read once.
AHB_DEVICE bool is_tiles(const Args& a, const Group& g) { return query_rows(a, g) > RT; }

// Units of the row kernel: 16 cache rows for all query rows of one key head.
AHB_DEVICE int row_units(const Group& g) { return ceil_div(g.keys, KU); }

// Units of the tile kernel for the rt-th pair of tiles: 64 cache rows against two tiles, or 128 against one.
// An item's first ITEM_COST units stand for its beginning and end, which take as long as that many blocks, and hold no block:
// thread blocks with many short items get as much to do as those with one long one.
constexpr int ITEM_COST = 4;
struct TileItem {
  int rows, blocks, units;  // valid query rows, blocks of cache rows that any of them sees, units with ITEM_COST
};
AHB_DEVICE TileItem tile_item(const Args& a, const Group& g, int rt) {
  const int G = a.H / a.Hk;
  TileItem t;
  t.rows = min(2 * a.tile_rows, g.tokens * G - 2 * a.tile_rows * rt);
  const int last = per_group(2 * a.tile_rows * rt + t.rows - 1, G);  // the last token
  t.blocks = ceil_div((int)min((int64_t)g.keys, (int64_t)g.before + last + 1), TK);
  t.units = ITEM_COST + (t.rows > a.tile_rows ? t.blocks : (t.blocks + 1) >> 1);
  return t;
}
AHB_DEVICE int row_tiles(const Args& a, const Group& g) { return ceil_div(query_rows(a, g), 2 * a.tile_rows); }

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

// Units of each of n workers: equal shares of all.
AHB_DEVICE int64_t share_of(int64_t units, int n) { return div64(units + n - 1, n); }

}  // namespace cattn
}  // namespace ahb
