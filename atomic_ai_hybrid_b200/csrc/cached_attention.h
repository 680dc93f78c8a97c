// What the kernels of cached attention share: the call's arguments and the plan that they work from.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace ahb {
namespace cattn {

using bf16 = __nv_bfloat16;

// One block of query rows and the cache rows that it sees: a sequence's own rows, or the rows of a prefix for
// the sequences of a run that share it.
struct Group {
  int row0, tokens;  // packed token rows row0 .. row0 + tokens (tokens 0: nothing to do)
  int slot, keys;    // cache slot, rows of it that any token sees
  int before;        // token t sees rows j <= before + t (a prefix: all of them)
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
  float scale2;                  // sm_scale log2(e)
  bf16* o;                       // (T, H, D)
  // workspace
  bf16* qw;                      // (T, H, D) rotated queries
  int* row_seq;                  // (T) sequence of a row, -1: none
  Group* groups;                 // [0, B) own rows, [B, 2 B) prefix runs at their last sequence
  int *run_start, *run_end;      // a sequence's run: its first sequence (-1: no prefix), and that one's last
  int64_t* units;                // exclusive sums of the groups' units: own (B + 1), runs (B + 1), mass (B + 1)
  float* lse;                    // (T, H) log2 of the softmax's denominators, for mass
  float* part;                   // partial results of items that several warps share, two a warp
  float* full;                   // (2, T, H, D + 2) whole results of own rows and of prefix rows, if there is a prefix
  int warps;                     // warps of the row kernel
};

}  // namespace cattn
}  // namespace ahb
