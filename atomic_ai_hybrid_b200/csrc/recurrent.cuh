// Shared by the stateful serving kernels (selective_scan.cu, gdn_recurrent.cu): sequence lookup,
// typed row access, the exponential of a decay, and the 4-tap convolution of one channel.
#pragma once
#include "common.cuh"

namespace ahb {

// Tokens [start, end) of sequence b.  Packed rows: cu[b] .. cu[b + 1], forced into [0, T] so that
// no offset a caller passes can lead outside the inputs; otherwise rows of L tokens each.
struct SeqRange { int start, end; };
AHB_DEVICE SeqRange seq_range(const int* cu, int b, int L, int T) {
  if (cu == nullptr) return {b * L, b * L + L};
  const int s = min(max(__ldg(cu + b), 0), T);
  return {s, min(max(__ldg(cu + b + 1), s), T)};
}

// Rows that no sequence covers, [0, cu[0]) and [cu[B], T).  Every block of a call with offsets clears some of them, so
// that no row of the output keeps what its memory held before.
struct OpenRows {
  int head, tail, count;
  AHB_DEVICE OpenRows(const int* cu, int B, int T) {
    head = min(max(__ldg(cu), 0), T);
    tail = min(max(__ldg(cu + B), head), T);
    count = head + T - tail;
  }
  AHB_DEVICE int row(int i) const { return i < head ? i : tail + i - head; }
};

// State slot of sequence b, -1 if it has none (a padding row): such rows give zeros, touch no state.
AHB_DEVICE int seq_slot(const int* slots, int b, int S) {
  const int s = slots ? __ldg(slots + b) : b;
  return s >= 0 && s < S ? s : -1;
}

// e^x for x <= 0 to about one unit in the last place: x = n ln 2 + r with ln 2 in two parts (Cody and
// Waite, 355/512 and the rest), Taylor in r to r^7 (|r| <= 0.347, remainder below 6e-9).  A decay multiplies the state
// once per token, so the 2^-22 error of the hardware's ex2 would add up over a state's memory.  Growth is right too:
// n ends at 127, the largest exponent, and r takes the rest up to infinity (2e-6 off at e^88.7, the floats' end).
AHB_DEVICE float exp_decay(float x) {
  x = fmaxf(x, -87.f);
  const float n = fminf(rintf(x * 1.4426950408889634f), 127.f);
  float r = fmaf(n, -355.f / 512.f, x);
  r = fmaf(n, 2.1219444005469e-4f, r);
  float p = fmaf(r, 1.f / 5040.f, 1.f / 720.f);
  p = fmaf(p, r, 1.f / 120.f);
  p = fmaf(p, r, 1.f / 24.f);
  p = fmaf(p, r, 1.f / 6.f);
  p = fmaf(p, r, 0.5f);
  p = fmaf(p, r, 1.f);
  p = fmaf(p, r, 1.f);
  return p * __int_as_float(((int)n + 127) << 23);
}

template <typename W>
AHB_DEVICE void load_taps(float w[4], const W* p) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = to_f(p[j]);
}

// SiLU of the causal 4-tap window (oldest first)
AHB_DEVICE float conv_silu(const float w[4], float bias, float x0, float x1, float x2, float x3) {
  float a = fmaf(w[0], x0, bias);
  a = fmaf(w[1], x1, a);
  a = fmaf(w[2], x2, a);
  return siluf_(fmaf(w[3], x3, a));
}

}  // namespace ahb
