// Arguments of the attention kernels for sequences of any length (csrc/mha.hip), shared with bindings.cpp.
// Plain host header: no HIP or torch types besides pointers.
#pragma once
#include <stdint.h>

enum { MHA_BF16 = 0, MHA_F16 = 1, MHA_F32 = 2 };

struct MhaArgs {
  const void *q, *k, *v;
  void* o;      // forward: written; backward: read
  float* lse;   // (B, H, Tq), natural log of the row's sum of exponentials; -inf where a row sees no key
  const void* dout;
  void *dq, *dk, *dv;
  float* delta;  // (2, B, H, Tq) workspace of the backward: rowsum(dO * O), then (float16) max |dO| of each row
  // workspace of sums over a split axis, joined by a further launch (see mta_mha_plan):
  //   forward (splits, B * Hkv, G * Tq, D + 2): unnormalised rows, running maximum and sum
  //   backward (dq_splits, B * Hkv, G * Tq, D), then (kv_splits, 2, B * Hkv, Tk, D): dK and dV
  float* part;
  const int* lens;  // (B) keys of each sequence, clamped to [0, Tk]; null: Tk
  // strides in elements: batch, token, head (the head dimension itself is contiguous)
  long qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];
  int B, Tq, Tk, H, Hkv, G, D;
  int causal;
  float scale;
  unsigned gmul, gshift;  // row / G = row * gmul >> gshift (set by mta_mha)
  int splits;       // forward: key ranges a row tile is split over
  int split_tiles;  // key tiles in each of them
  int dq_splits, dq_split_tiles;  // the same of the dQ kernel
  int kv_splits;    // row ranges a key tile is split over (dK, dV kernel)
};

// elements of a tensor with 4 dimensions: `at` of the first, strides and sizes, in elements
struct MhaBox {
  long at, strides[4], sizes[4];
};
