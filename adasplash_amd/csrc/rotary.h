// Positions of queries and keys: what the C entry points (rotary.hip) hand to the kernels of one element type (rotary_unit.hip).
#pragma once
#include "common.h"

namespace adsp {
namespace rotary {
constexpr int kThreads = 256;

// Rows of one tensor of heads; strides in elements: batch item, head, token.
struct Rows {
  const void *x, *dy;
  void* y;  // turned rows, or the gradient of x
  const void* weight;  // [D] of a norm, or null: no norm
  float* partial;      // of the weight's gradient: [workgroups][D]
  long long x_b, x_h, x_n, y_b, y_h, y_n, dy_b, dy_h, dy_n;
  int heads, blocks;  // blocks: workgroups along the heads
};
struct Pages {
  const long long* slots;
  const char* v;
  char* v_pages;
  long long v_st, v_sh, k_sp, k_sph, k_sps, v_sp, v_sph, v_sps;  // bytes; k's pages take Rows::y
  long long n_slots;
  int page;
};
struct Params {
  Rows of[2];  // q, k
  Pages pages;
  const void* positions;
  const double* frequencies;
  long long pos_b, pos_n;
  uint32_t tokens, N;  // tokens: B * N, below 2^31 less a workgroup's
  int pos_bits, weight_f32[2];
  int rot, per;  // per: heads that a workgroup takes
  int token_blocks, token_steps;
  float eps, factor, inv_d;
};

// Launchers of one element type.  mode 0: rows to rows, 1: rows to the slots of pages, 2: gradients.
template <typename T> void launch(const Params& p, int D, bool half, int mode, hipStream_t s);
}  // namespace rotary
}  // namespace adsp
