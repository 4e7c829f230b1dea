// What grouped.cu and grouped_few.cu share, and what the first hands to the second.
#ifndef SPARSETIR_B200_GROUPED_H_
#define SPARSETIR_B200_GROUPED_H_

#include "common.h"
#include "launch.cuh"

namespace sptir {

// The last of the groups that starts at or before the row, group 0 if none does: 32 pointers at a time, by all lanes of a warp
// together.
__device__ __forceinline__ int group_of_row(const int32_t* indptr, int groups, long long row, int lane) {
  int lo = 0, n = groups;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const bool in = lane * step < n && ld_global(indptr + lo + min(lane * step, n - 1)) <= row;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, in) | 1u);
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

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
