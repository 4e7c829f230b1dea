// Products of a feed-forward block grouped by expert, beyond the plain ones of grouped.cu:
//   grouped_mm_gated       h = x W[g]^T of 2 * width features, act = f(h[:, :width]) * h[:, width:]  (gate.cuh)
//   grouped_mm_gated_grad  d_act = dy W[g], and from it and h the gradient to h
//   grouped_mm_f8, grouped_mm_gated_f8  of 8-bit floating point (e4m3) with a scale for each 128 of a row of x and each 128 x 128 of W
// In their simplest form: 32 x 32 results to a block, operands through shared memory, sums in f32 on the CUDA cores.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.h"
#include "gate.cuh"
#include "grouped.h"
#include "launch.cuh"
#include "lowp.cuh"

namespace sptir {

__device__ __forceinline__ float to_float(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

namespace {

constexpr int kT = 32;
constexpr int kScaleBlock = 128;  // elements that share a scale

struct Shape {
  const int32_t* indptr;
  int rows, groups, k, feats;
};

// x and W in one type, W of `wide` rows of k elements, or with along_k false k rows of `wide`.
template <class T>
struct Operands {
  const T* x;
  const T* w;
  const float* x_scale;  // [blocks][rows], null: none
  const float* w_scale;  // [groups][blocks of rows][blocks]
  int wide, along_k;
  __device__ __forceinline__ float x_at(const Shape& s, int row, int k) const {
    const float v = to_float(x[static_cast<size_t>(row) * s.k + k]);
    return x_scale != nullptr ? v * x_scale[static_cast<size_t>(k / kScaleBlock) * s.rows + row] : v;
  }
  __device__ __forceinline__ float w_at(const Shape& s, int group, int f, int k) const {
    const size_t at = along_k ? (static_cast<size_t>(group) * wide + f) * s.k + k : (static_cast<size_t>(group) * s.k + k) * wide + f;
    const float v = to_float(w[at]);
    if (w_scale == nullptr) return v;
    const int fb = (wide + kScaleBlock - 1) / kScaleBlock, kb = (s.k + kScaleBlock - 1) / kScaleBlock;
    return v * w_scale[(static_cast<size_t>(group) * fb + f / kScaleBlock) * kb + k / kScaleBlock];
  }
};

template <class OutT>
struct StorePlain {
  static constexpr bool kTwo = false;
  OutT* y;
  __device__ __forceinline__ void operator()(const Shape& s, int row, int f, float v, float) const {
    y[static_cast<size_t>(row) * s.feats + f] = from_float<OutT>(v);
  }
};
template <class T>
struct StoreGated {
  static constexpr bool kTwo = true;
  T* y;
  T* hidden;
  Gate gate;
  __device__ __forceinline__ void operator()(const Shape& s, int row, int f, float g, float up) const {
    y[static_cast<size_t>(row) * s.feats + f] = from_float<T>(gate.act(g, up));
    if (hidden != nullptr) {
      T* h = hidden + static_cast<size_t>(row) * 2 * s.feats + f;
      h[0] = from_float<T>(g);
      h[s.feats] = from_float<T>(up);
    }
  }
};
template <class T>
struct StoreGrad {
  static constexpr bool kTwo = false;
  const T* hidden;
  T* d_hidden;
  T* act;
  Gate gate;
  __device__ __forceinline__ void operator()(const Shape& s, int row, int f, float d, float) const {
    const size_t at = static_cast<size_t>(row) * 2 * s.feats + f;
    float dg, du, a;
    gate.grad(to_float(hidden[at]), to_float(hidden[at + s.feats]), d, &dg, &du, &a);
    d_hidden[at] = from_float<T>(dg);
    d_hidden[at + s.feats] = from_float<T>(du);
    if (act != nullptr) act[static_cast<size_t>(row) * s.feats + f] = from_float<T>(a);
  }
};

// Block: 32 rows from 32 blockIdx.y on, 32 features; the groups that the rows belong to, one after the other.
template <class T, class Store>
__global__ void __launch_bounds__(256) block_kernel(Shape s, Operands<T> op, Store store) {
  constexpr bool kTwo = Store::kTwo;
  __shared__ float xs[kT][kT + 1], ws[kTwo ? 2 : 1][kT][kT + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int f0 = blockIdx.x * kT, r0 = blockIdx.y * kT;
  int group = s.indptr != nullptr ? group_of_row(s.indptr, s.groups, r0, tx) : 0;
  for (; group < s.groups; ++group) {
    const int first = s.indptr != nullptr ? min(max(s.indptr[group], 0), s.rows) : 0;
    const int last = s.indptr != nullptr ? min(s.indptr[group + 1], s.rows) : s.rows;
    if (first >= r0 + kT) break;
    if (last <= r0 || last <= first) continue;
    float acc[2][4] = {};
    for (int k0 = 0; k0 < s.k; k0 += kT) {
      __syncthreads();
      for (int i = ty; i < kT; i += 8) {
        const int k = k0 + tx;
        xs[i][tx] = r0 + i >= first && r0 + i < last && k < s.k ? op.x_at(s, r0 + i, k) : 0.f;
#pragma unroll
        for (int h = 0; h < (kTwo ? 2 : 1); ++h)
          ws[h][i][tx] = f0 + i < s.feats && k < s.k ? op.w_at(s, group, f0 + i + h * s.feats, k) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kT; ++k)
#pragma unroll
        for (int h = 0; h < (kTwo ? 2 : 1); ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[h][i] = fmaf(xs[ty + 8 * i][k], ws[h][tx][k], acc[h][i]);
    }
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + ty + 8 * i;
      if (row >= first && row < last && f0 + tx < s.feats) store(s, row, f0 + tx, acc[0][i], acc[1][i]);
    }
  }
}

template <class T, class Store>
int launch(const Shape& s, const Operands<T>& op, const Store& store, cudaStream_t st) {
  const dim3 grid(ceil_div(s.feats, kT), ceil_div(s.rows, kT));
  block_kernel<T, Store><<<grid, 256, 0, st>>>(s, op, store);
  SPTIR_LAUNCH_OK("block_kernel");
  return 0;
}

int check(const char* fn, const int32_t* indptr, int rows, int groups, int fi, int fo, bool twice, int flags, int known) {
  if (rows < 0 || groups < 0) return fail("%s: negative size", fn);
  if (fi < 1 || fo < 1) return fail("%s: feat_in and %s must be positive", fn, twice ? "width" : "feat_out");
  if (std::max(std::max(rows, groups), std::max(fi, fo)) > kLargestSize || (twice && fo > kLargestSize / 2) ||
      (groups > 0 && static_cast<long long>(fi) * fo * (twice ? 2 : 1) > INT64_MAX / groups))
    return fail("%s: too large for 32-bit indices", fn);
  if ((flags & ~known) != 0) return fail("%s: unknown flags %d", fn, flags);
  if (!indptr && groups > 1) return fail("%s: indptr may be null with num_groups 1 only", fn);
  return 0;
}
int check_pointers(const char* fn, const int32_t* indptr, int rows, int groups, cudaStream_t st) {
  if (!indptr || !validate_enabled()) return 0;
  if (validate_indptr(fn, "indptr", indptr, groups, -1, st) != 0) return -1;
  return validate_range(fn, "indptr", indptr, groups + 1ll, rows + 1ll, st);
}

// f(T{}) for the 16-bit type
template <class F>
int with_half(int type, F&& f) {
  if (type == SPARSETIR_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace
}  // namespace sptir

using namespace sptir;

extern "C" int sparsetir_grouped_mm_gated_raw(const void* x, const void* w, void* y, void* hidden, int type, const int32_t* indptr,
                                              int rows, int num_groups, int feat_in, int width, int flags, int device_id,
                                              void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated";
  if (check(fn, indptr, rows, num_groups, feat_in, width, true, flags, SPARSETIR_GATED_GELU) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: x, w, y and hidden are f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !w || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const Operands<T> op{static_cast<const T*>(x), static_cast<const T*>(w), nullptr, nullptr, 2 * width, 1};
    return launch(Shape{indptr, rows, num_groups, feat_in, width}, op,
                  StoreGated<T>{static_cast<T*>(y), static_cast<T*>(hidden), Gate((flags & SPARSETIR_GATED_GELU) != 0)}, st);
  });
}

extern "C" int sparsetir_grouped_mm_gated_grad_raw(const void* dy, const void* w, const void* hidden, void* d_hidden, void* act,
                                                   int type, const int32_t* indptr, int rows, int num_groups, int feat, int width,
                                                   int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated_grad";
  if (check(fn, indptr, rows, num_groups, feat, width, true, flags, SPARSETIR_GATED_GELU | SPARSETIR_GROUPED_W_OUT_IN) != 0) return -1;
  if (type != SPARSETIR_F16 && type != SPARSETIR_BF16) return fail("%s: all tensors are f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!dy || !w || !hidden || !d_hidden) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const Operands<T> op{static_cast<const T*>(dy), static_cast<const T*>(w), nullptr, nullptr, width,
                         (flags & SPARSETIR_GROUPED_W_OUT_IN) != 0};
    return launch(Shape{indptr, rows, num_groups, feat, width}, op,
                  StoreGrad<T>{static_cast<const T*>(hidden), static_cast<T*>(d_hidden), static_cast<T*>(act),
                               Gate((flags & SPARSETIR_GATED_GELU) != 0)}, st);
  });
}

extern "C" int sparsetir_grouped_mm_f8_raw(const void* x, const float* x_scale, const void* w, const float* w_scale, void* y, int y_type,
                                           const int32_t* indptr, int rows, int num_groups, int feat_in, int feat_out, int device_id,
                                           void* stream) {
  const char* fn = "sparsetir_grouped_mm_f8";
  if (check(fn, indptr, rows, num_groups, feat_in, feat_out, false, 0, 0) != 0) return -1;
  if (y_type < SPARSETIR_F32 || y_type > SPARSETIR_BF16) return fail("%s: unknown element type %d", fn, y_type);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_type(y_type, [&](auto o) {
    using O = decltype(o);
    const Operands<__nv_fp8_e4m3> op{static_cast<const __nv_fp8_e4m3*>(x), static_cast<const __nv_fp8_e4m3*>(w), x_scale, w_scale, feat_out, 1};
    return launch(Shape{indptr, rows, num_groups, feat_in, feat_out}, op, StorePlain<O>{static_cast<O*>(y)}, st);
  });
}

extern "C" int sparsetir_grouped_mm_gated_f8_raw(const void* x, const float* x_scale, const void* w, const float* w_scale, void* y,
                                                 int y_type, const int32_t* indptr, int rows, int num_groups, int feat_in, int width,
                                                 int flags, int device_id, void* stream) {
  const char* fn = "sparsetir_grouped_mm_gated_f8";
  if (check(fn, indptr, rows, num_groups, feat_in, width, true, flags, SPARSETIR_GATED_GELU) != 0) return -1;
  if (y_type != SPARSETIR_F16 && y_type != SPARSETIR_BF16) return fail("%s: y is f16 or bf16", fn);
  if (rows == 0 || num_groups == 0) return 0;
  if (!x || !x_scale || !w || !w_scale || !y) return fail("%s: null pointer argument", fn);
  if (use_device(device_id) != 0) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (check_pointers(fn, indptr, rows, num_groups, st) != 0) return -1;
  return with_half(y_type, [&](auto t) {
    using T = decltype(t);
    const Operands<__nv_fp8_e4m3> op{static_cast<const __nv_fp8_e4m3*>(x), static_cast<const __nv_fp8_e4m3*>(w), x_scale, w_scale, 2 * width, 1};
    return launch(Shape{indptr, rows, num_groups, feat_in, width}, op,
                  StoreGated<T>{static_cast<T*>(y), nullptr, Gate((flags & SPARSETIR_GATED_GELU) != 0)}, st);
  });
}
