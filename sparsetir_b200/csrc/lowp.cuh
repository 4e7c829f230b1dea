// Elements of the operators that take f32, f16 and bf16: pieces of 2 to 16 bytes as floats and back.  Every sum is formed
// in f32; a result is rounded once, to nearest even, when it is packed.
#ifndef SPARSETIR_B200_LOWP_CUH_
#define SPARSETIR_B200_LOWP_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sparsetir_b200.h"

namespace sptir {

template <int BYTES> struct PieceOf;
template <> struct PieceOf<16> { using type = uint4; };
template <> struct PieceOf<8> { using type = uint2; };
template <> struct PieceOf<4> { using type = uint32_t; };
template <> struct PieceOf<2> { using type = uint16_t; };
template <> struct PieceOf<1> { using type = uint8_t; };
template <int BYTES> using Piece = typename PieceOf<BYTES>::type;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A piece of BYTES bytes as the floats of its elements
template <class T, int BYTES>
__device__ __forceinline__ void unpack(const Piece<BYTES>& p, float (&f)[BYTES / sizeof(T)]) {
  const T* t = reinterpret_cast<const T*>(&p);
#pragma unroll
  for (int i = 0; i < BYTES / static_cast<int>(sizeof(T)); ++i) f[i] = to_float(t[i]);
}
template <class T, int BYTES>
__device__ __forceinline__ Piece<BYTES> pack(const float (&f)[BYTES / sizeof(T)]) {
  Piece<BYTES> p;
  T* t = reinterpret_cast<T*>(&p);
#pragma unroll
  for (int i = 0; i < BYTES / static_cast<int>(sizeof(T)); ++i) t[i] = from_float<T>(f[i]);
  return p;
}

// f(T{}) for the element type `type` (SPARSETIR_F32 / F16 / BF16)
template <class F>
inline int with_type(int type, F&& f) {
  if (type == SPARSETIR_F32) return f(float{});
  if (type == SPARSETIR_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace sptir
#endif  // SPARSETIR_B200_LOWP_CUH_
