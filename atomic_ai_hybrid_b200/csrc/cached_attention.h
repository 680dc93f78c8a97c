// What the kernels of cached attention share: the call's arguments and the plan that they work from.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace ahb {
namespace cattn {

using bf16 = __nv_bfloat16;

// A block of query rows and the cache rows that they see: a sequence's own rows, or the rows of a prefix for
// the sequences of a run that share it.
struct Group {
  int row0, tokens;  // packed token rows row0 .. row0 + tokens (tokens 0: nothing to do)
  int slot, keys;    // cache slot, rows of it that any token sees
  int before;        // token t sees rows j < min(keys, before + t + 1) (a prefix: before = keys)
  int64_t per_head;  // units of a key head, in the kernel that takes the group
};

// Groups [0, B) are the sequences' own rows, [B, 2 B) the prefix runs, each at its last sequence.  Each group is worked on by one of
// two kernels; a kernel's units are numbered through the groups, and sums[kind][g] is group g's first one.
enum Kind { ROWS = 0, TILES = 1, TILES_MASS = 2, KINDS = 3 };

// What a block of the tile kernel began and others go on with (rows 0: nothing), up to block `last`.
struct SharedItem {
  int row0, r0, rows, h, last;
};

struct Args {
  const bf16 *q, *k, *v;
  int64_t qs, ks, vs;            // row strides
  bf16 *kc, *vc;                 // (S, Hk, M, D)
  const int *lengths, *seen, *slots, *cu, *prefix;
  const float *cos, *sin;
  int table;                     // rows of the tables, -1: no rotation
  int B, L, T, S, M, H, Hk, D;
  float* mass;
  int* held;
  float scale2;                  // sm_scale log2(e), without its sign
  bool negate;                   // the sign: the rotated queries are negated
  // Exponents are s scale2 - m, in the tile kernel and for its masses by one fused operation: the product is exact there and rounded in
  // m, so that all of a row's weights and their sum carry one factor, up to 2^(half a step of m), and a quotient none.  Where scores can
  // pass 2^28 that factor could leave 32 bits: there the product is rounded before too, with a product and a sum for each exponent (2407
  // tokens on 4100 shared rows at the scales 1.4 and 1.5, fused and rounded: 278 and 290 us, a prompt of 8192 613 and 610).
  bool rounded;
  bf16* o;                       // (T, H, D)
  // workspace
  bf16* qw;                      // (T, H, 2, D) rotated queries rounded to bf16, and what the rounding left of them
  int* row_seq;                  // (T) sequence of a row, -1: none
  Group* groups;                 // (2 B)
  int *run_start, *run_end;      // a sequence's run: its first sequence (-1: no prefix), and that one's last
  int64_t* sums[KINDS];          // (2 B + 1) each
  float* scores;                 // the row kernel's, unit by unit (8 query rows of 16 cache rows), for mass
  float2* lse;                   // (T, H) the softmax's maximum, as an exponent of 2, and one over its denominator, for mass
  float* part;                   // partial results of items that several warps share, two a warp
  float* tile_part;              // ... of items that several blocks share, two a block
  SharedItem* shared_items;      // (blocks)
  int64_t* shares;               // units of a worker of the row kernel and of the tile kernel
  float* full;                   // (2, T, H, D + 4) whole results of own rows and of prefix rows, if there is a prefix
  int tile_rows;                 // query rows of a tile: as many tokens as fit into 128 rows, with their heads
  int warps, blocks;             // warps of the row kernel, blocks of the tile kernel (0: it is not launched)
  int* err;                      // error word of waits that ran out
};

// The tile kernel (cached_attention_tc.cu).
int launch_tiles(const Args& a, cudaStream_t st);

}  // namespace cattn
}  // namespace ahb
