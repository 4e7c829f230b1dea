// The gate of a feed-forward block: act = f(gate) * up with f(g) = g * sigmoid(z(g)),
//   silu                z = g
//   gelu, form of tanh  0.5 g (1 + tanh(u)) = g * sigmoid(2 u):  z = 2 sqrt(2 / pi) (g + 0.044715 g^3)
// and its gradient: with s = sigmoid(z),  f' = s + g s (1 - s) z'.
// All of it in f32; exp and the quotient by the hardware's approximations (a few units of 2^-22: nothing beside the rounding of a 16-bit
// result, and z is at most 88 in magnitude where s is not 0 or 1 to that precision).
#ifndef SPARSETIR_B200_GATE_CUH_
#define SPARSETIR_B200_GATE_CUH_

#include <cuda_runtime.h>

namespace sptir {

struct Gate {
  float c1 = 1.f, c3 = 0.f;  // z = g (c1 + c3 g^2)
  Gate() = default;
  explicit Gate(bool gelu) {
    if (gelu) {
      c1 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
      c3 = 0.07135481282652936f;  // and times 0.044715
    }
  }
  __device__ __forceinline__ float sigmoid(float g, float g2) const {
    return __fdividef(1.f, 1.f + __expf(-g * fmaf(c3, g2, c1)));  // exp is infinite from about 88 on: 1 / inf = 0
  }
  // bounded: c3 = 0 times an infinite square would not be a number
  static __device__ __forceinline__ float square(float g) { return fminf(g * g, 1e30f); }
  __device__ __forceinline__ float act(float g, float up) const { return g * sigmoid(g, square(g)) * up; }
  // d: gradient of act
  __device__ __forceinline__ void grad(float g, float up, float d, float* d_gate, float* d_up, float* act) const {
    const float g2 = square(g), s = sigmoid(g, g2), f = g * s;
    *d_gate = d * up * fmaf(f * (1.f - s), fmaf(3.f * c3, g2, c1), s);
    *d_up = d * f;
    *act = f * up;
  }
};

}  // namespace sptir
#endif  // SPARSETIR_B200_GATE_CUH_
