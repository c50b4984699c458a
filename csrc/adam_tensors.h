// Argument table of the Adam / AdamW step over many tensors (csrc/adam_tensors.hip), shared with bindings.cpp.
#pragma once
#include <stdint.h>

constexpr int ADAM_BLOCK = 256;   // elements of a tensor that share one power of two (8-bit moments)
constexpr long ADAM_GROUPS = 0xffffff;  // workgroups of one launch: of 256 threads, and a launch holds 2^32 - 1
constexpr int ADAM_TABLE = 112;   // tensors of one launch: the table travels by value, as kernel arguments (< 4 KB)

// element types of a tensor and its gradient: p | g << 2
enum { ADAM_F32 = 0, ADAM_BF16 = 1, ADAM_F16 = 2 };

struct AdamTable {
  void* p[ADAM_TABLE];
  void* g[ADAM_TABLE];
  long n[ADAM_TABLE];               // elements; 0 for a tensor that is left out of the step
  unsigned block[ADAM_TABLE];       // first block of its moments
  unsigned first[ADAM_TABLE];       // first workgroup of the launch that takes it
  unsigned char type[ADAM_TABLE];
  int count;
  int place;                        // of the table's first tensor among the optimizer's
  int group;                        // elements of a workgroup
  unsigned groups;                  // workgroups over all tensors
};

struct AdamState {
  float* m32;          // 32-bit moments: blocks of 256 values
  float* v32;
  unsigned char* m8;   // 8-bit moments: blocks of 256 codes
  unsigned char* v8;
  signed char* em;     // a block's power of two
  signed char* ev;
  const float* lr;
  float* step;         // steps taken
  float* steps;        // steps that each of the optimizer's `count` tensors has taken
  float* factors;      // each tensor's factors of this step, four floats (see ADAM_F_*)
  double* parts;       // norm partials
  unsigned* ticket;
  float* ctl;          // this step's factors (see ADAM_CTL_*)
  float* norm;
  float* nonfinite;
  uint64_t seed;
  float beta1, beta2, one_beta1, one_beta2, eps, wd;
  double dbeta1, dbeta2, dwd, max_norm, scale;
  int decoupled, zero_grad, count;
  int skip;            // a step whose gradient norm is not finite changes nothing (the norm is taken without clipping too)
};
