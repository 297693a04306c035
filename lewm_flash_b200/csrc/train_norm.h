// Layer norm and adaptive layer norm: arguments of the kernels, and their launch per element type.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lewm {

struct NormArgs {
  const void* x;
  const void* dy;
  const void* a;       // weight or scale, or null (a = 1)
  const void* b;       // bias or shift, or null
  void* out;           // y or dx
  float* stats;        // [2][rows]: mu, rs
  void* da;            // [groups][width] in the parameters' type, or null
  void* db;
  float* ws;           // [groups * split][2][width] partial sums when split > 1
  int64_t rows, x_stride, dy_stride, a_stride, b_stride;
  int64_t group;       // rows per (a, b)
  int64_t items;       // groups * split
  int split;           // items per group
  int loop_min, loop_rem;  // a loop that starts `o` rows into its rows has loop_min + (o < loop_rem) rounds
  int width;
  int p_type;
  int one_plus;        // a = 1 + a[]
  int team_items;      // 1: an item per team, 0: per block
  int stages;          // of the ring
  int p_vec;           // 1: E parameters load as vectors
  float eps;
};

// Launches one pass over rows of T (float, __nv_bfloat16, __half; a translation unit each) without the
// final reduction of partial sums. `wide`: rows of more than kMaxRowBytes; `vec`: bytes of the vectors
// that all rows start on (16, 8, 4 or one element's).
template <typename T>
cudaError_t launch_norm_rows(const NormArgs& p, bool wide, bool backward, int vec, cudaStream_t st);

constexpr int kSms = 148;              // B200
constexpr int kMaxRowBytes = 32768;    // widest row held by a block: 512 threads x 32 16-bit elements

}  // namespace lewm
