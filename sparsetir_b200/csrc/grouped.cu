// Products grouped by expert, ragged sizes: the simplest form that is right for every size, on CUDA cores.
#include <algorithm>

#include "common.h"
#include "launch.cuh"
#include "lowp.cuh"

namespace sptir {
namespace {

constexpr int kTile = 64, kStep = 16;

// First and past the last row of group g, inside the array whatever the pointers say.
__device__ __forceinline__ void group_rows(const int32_t* indptr, int g, int rows, int* first, int* last) {
  if (indptr == nullptr) { *first = 0; *last = rows; return; }
  *first = min(max(ld_global(indptr + g), 0), rows);
  *last = max(min(ld_global(indptr + g + 1), rows), *first);
}

__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__half v) { return __half2float(v); }
__device__ __forceinline__ float number(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ int number(int8_t v) { return v; }

template <class T> struct SumOf { using type = float; };
template <> struct SumOf<int8_t> { using type = int; };

// c[64 x 64] += a[64 x 16] * b[16 x 64] out of shared memory, 4 x 4 results to a thread
template <class S>
__device__ __forceinline__ void multiply(S (&c)[4][4], const S (&a)[kStep][kTile + 1], const S (&b)[kStep][kTile + 1]) {
  const int r = threadIdx.x / 16, q = threadIdx.x % 16;
#pragma unroll
  for (int k = 0; k < kStep; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[i][j] += a[k][r + 16 * i] * b[k][q + 16 * j];
}

// Block = 64 features of 64 rows of one group; blockIdx.y counts the row tiles of all groups.
template <class T, class OutT>
__global__ void __launch_bounds__(256)
grouped_kernel(const T* x, const T* w, OutT* y, const float* x_scale, const float* w_scale, const int32_t* indptr, int rows,
               int groups, int fi, int fo, int out_in) {
  using S = typename SumOf<T>::type;
  __shared__ S a[kStep][kTile + 1], b[kStep][kTile + 1];
  chain_wait();
  int tile = blockIdx.y, g = 0, first = 0, last = 0;
  for (; g < groups; ++g) {
    group_rows(indptr, g, rows, &first, &last);
    const int n = (last - first + kTile - 1) / kTile;
    if (tile < n) break;
    tile -= n;
  }
  if (g == groups) return;
  first += tile * kTile;
  const int f0 = blockIdx.x * kTile;
  S c[4][4] = {};
  const T* wg = w + static_cast<size_t>(g) * fi * fo;
  for (int k0 = 0; k0 < fi; k0 += kStep) {
    for (int e = threadIdx.x; e < kStep * kTile; e += 256) {
      const int k = e % kStep, i = e / kStep;
      a[k][i] = 0;
      if (first + i < last && k0 + k < fi) a[k][i] = number(x[static_cast<size_t>(first + i) * fi + k0 + k]);
      b[k][i] = 0;
      if (f0 + i < fo && k0 + k < fi)
        b[k][i] = number(out_in ? wg[static_cast<size_t>(f0 + i) * fi + k0 + k] : wg[static_cast<size_t>(k0 + k) * fo + f0 + i]);
    }
    __syncthreads();
    multiply(c, a, b);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = first + threadIdx.x / 16 + 16 * i, f = f0 + threadIdx.x % 16 + 16 * j;
      if (r >= last || f >= fo) continue;
      float v = static_cast<float>(c[i][j]);
      if (x_scale != nullptr) v *= x_scale[r] * w_scale[static_cast<size_t>(g) * fo + f];
      y[static_cast<size_t>(r) * fo + f] = from_float<OutT>(v);
    }
}

// Block = 64 x 64 of one group's dw: the sum over the group's rows of a[s, i] * b[s, j]
template <class T, class OutT>
__global__ void __launch_bounds__(256)
grouped_grad_kernel(const T* pa, const T* pb, OutT* dw, const int32_t* indptr, int rows, int fa, int fb) {
  __shared__ float a[kStep][kTile + 1], b[kStep][kTile + 1];
  chain_wait();
  const int g = blockIdx.z, i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
  int first = 0, last = 0;
  group_rows(indptr, g, rows, &first, &last);
  float c[4][4] = {};
  for (int s0 = first; s0 < last; s0 += kStep) {
    for (int e = threadIdx.x; e < kStep * kTile; e += 256) {
      const int i = e % kTile, k = e / kTile;
      a[k][i] = 0.f;
      b[k][i] = 0.f;
      if (s0 + k < last && i0 + i < fa) a[k][i] = number(pa[static_cast<size_t>(s0 + k) * fa + i0 + i]);
      if (s0 + k < last && j0 + i < fb) b[k][i] = number(pb[static_cast<size_t>(s0 + k) * fb + j0 + i]);
    }
    __syncthreads();
    multiply(c, a, b);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = i0 + threadIdx.x / 16 + 16 * i, f = j0 + threadIdx.x % 16 + 16 * j;
      if (r < fa && f < fb) dw[(static_cast<size_t>(g) * fa + r) * fb + f] = from_float<OutT>(c[i][j]);
    }
}

int check_groups(const char* fn, const int32_t* indptr, int rows, int groups, int fi, int fo, int flags) {
  if (rows < 0 || groups < 0) return fail("%s: negative size", fn);
  if (fi < 1 || fo < 1) return fail("%s: feat_in and feat_out must be positive", fn);
  if ((flags & ~SPARSETIR_GROUPED_W_OUT_IN) != 0) return fail("%s: unknown flags %d", fn, flags);
  if (!indptr && groups > 1) return fail("%s: indptr may be null with num_groups 1 only", fn);
  return 0;
}
int check_pointers(const char* fn, const int32_t* indptr, int rows, int groups, cudaStream_t st) {
  if (!indptr || !validate_enabled()) return 0;
  if (validate_indptr(fn, "indptr", indptr, groups, -1, st) != 0) return -1;
  return validate_range(fn, "indptr", indptr, groups + 1ll, rows + 1ll, st);
}

template <class T, class OutT>
int run(const T* x, const T* w, OutT* y, const float* xs, const float* ws, const int32_t* indptr, int rows, int groups, int fi,
        int fo, int out_in, cudaStream_t st) {
  const dim3 grid(ceil_div(fo, kTile), ceil_div(rows, kTile) + groups);
  launch_chained(grouped_kernel<T, OutT>, grid, 256, 0, st, x, w, y, xs, ws, indptr, rows, groups, fi, fo, out_in);
  SPTIR_LAUNCH_OK("grouped_kernel");
  return 0;
}

}  // namespace
}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_grouped_mm_raw(const void* x, const void* w, int type, void* y, int y_type, const int32_t* indptr,
                                        int rows, int num_groups, int feat_in, int feat_out, int flags, int device_id,
                                        void* stream) {
  const char* fn = "sparsetir_grouped_mm";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, flags) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x and w are f16 or bf16", fn);
  if (y_type != type && y_type != SPARSETIR_F32) return fail("%s: y has the type of x, or f32", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !w || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return with_type(y_type, [&](auto o) {
      using O = decltype(o);
      return run(static_cast<const T*>(x), static_cast<const T*>(w), static_cast<O*>(y), nullptr, nullptr, indptr, rows, num_groups,
                 feat_in, feat_out, flags & SPARSETIR_GROUPED_W_OUT_IN, st);
    });
  });
}

extern "C" int sparsetir_grouped_mm_grad_w_raw(const void* x, const void* dy, int type, void* dw, int dw_type,
                                               const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out,
                                               int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_grad_w";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, flags) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x and dy are f16 or bf16", fn);
  if (dw_type != type && dw_type != SPARSETIR_F32) return fail("%s: dw has the type of x, or f32", fn);
  if (num_groups == 0) return 0;
  if (!dw || (rows > 0 && (!x || !dy))) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  const bool out_in = (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0;
  const int fa = out_in ? feat_out : feat_in, fb = out_in ? feat_in : feat_out;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return with_type(dw_type, [&](auto o) {
      using O = decltype(o);
      const dim3 grid(ceil_div(fb, kTile), ceil_div(fa, kTile), num_groups);
      launch_chained(grouped_grad_kernel<T, O>, grid, 256, 0, st, static_cast<const T*>(out_in ? dy : x),
                     static_cast<const T*>(out_in ? x : dy), static_cast<O*>(dw), indptr, rows, fa, fb);
      SPTIR_LAUNCH_OK("grouped_grad_kernel");
      return 0;
    });
  });
}

extern "C" int sparsetir_grouped_mm_i8_raw(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, void* y,
                                           int y_type, const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out,
                                           int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_i8";
  if (check_groups(fn, indptr, rows, num_groups, feat_in, feat_out, 0) != 0) return -1;
  if (feat_in >= 131072) return fail("%s: feat_in = %d: sums of more than 131071 products may not fit 32 bits", fn, feat_in);
  if (y_type < SPARSETIR_F32 || y_type > SPARSETIR_BF16) return fail("%s: unknown element type %d", fn, y_type);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_type(y_type, [&](auto o) {
    using O = decltype(o);
    return run(x, w, static_cast<O*>(y), x_scale, w_scale, indptr, rows, num_groups, feat_in, feat_out, 1, st);
  });
}
