// What grouped.cu hands to grouped_few.cu.
#ifndef SPARSETIR_B200_GROUPED_H_
#define SPARSETIR_B200_GROUPED_H_

#include "common.h"

namespace sptir {

struct FewArgs {
  const void* x;
  const void* w;
  void* y;
  const float* x_scale;
  const float* w_scale;
  const int32_t* indptr;
  size_t x_pitch, w_pitch;  // bytes of a row, multiples of 16
  int rows, groups, fi, fo;
  int k_bytes;              // of a row of x
  int splits, split_bytes, feature_warps;  // set by the launcher
};

// y = x * W by the kernel for groups of a few rows; `type` as SPARSETIR_F16 / BF16, -1 for 8-bit integers; along_k: W is
// contiguous along the depth.
int few_rows(const FewArgs& p, int type, int y_type, bool along_k, cudaStream_t st);

}  // namespace sptir
#endif  // SPARSETIR_B200_GROUPED_H_
