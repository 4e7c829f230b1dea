// The gate of a feed-forward block: act = f(gate) * up with f(g) = g * sigmoid(z(g)),
//   silu                z = g
//   gelu, form of tanh  0.5 g (1 + tanh(u)) = g * sigmoid(2 u):  z = 2 sqrt(2 / pi) (g + 0.044715 g^3)
// and its gradient: with s = sigmoid(z),  f' = s + g s (1 - s) z'.
// All of it in f32; exp and the quotient by the hardware's approximations.  The exponential multiplies the few roundings of its argument by |z|:
// f and act are off by (8 |z| + 32) 2^-24 of their value at most, 2^-14 where they are still above 2^-140 (|z| = 104).  That is little beside the
// rounding of a 16-bit result; one of 32 bits would show it.
#ifndef SPARSETIR_B200_GATE_CUH_
#define SPARSETIR_B200_GATE_CUH_

#include <cuda_runtime.h>

#include <cstdint>

namespace sptir {

// Two floats that go through one instruction, half as many of them to issue in the epilogues of the products.  (Us, floats one by one / this, two
// runs each: gated products of 6,001 rows 73.4 73.6 / 73.0 73.2, of 65,536 rows 463 463 / 462 462, the gradient 320 361 / 322 317, in 8-bit
// floating point 186 182 / 179 184.)
struct Two {
  uint64_t v;
  Two() = default;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ float lo() const { return __uint_as_float(static_cast<uint32_t>(v)); }
  __device__ __forceinline__ float hi() const { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
  __device__ __forceinline__ friend Two operator*(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
  }
  __device__ __forceinline__ friend Two operator+(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
  }
};
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {  // a b + c
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float exp2_near(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));  // without ftz: results down to 2^-149
  return r;
}
__device__ __forceinline__ float reciprocal_near(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct Gate {
  bool gelu = false;
  static constexpr float kC1 = 1.5957691216057308f;   // 2 sqrt(2 / pi)
  static constexpr float kC3 = 0.07135481282652936f;  // and times 0.044715
  Gate() = default;
  explicit Gate(bool g) : gelu(g) {}

  // An infinite square would make z' g s (1 - s) = inf * 0.
  __device__ __forceinline__ static Two square(Two g) {
    const Two q = g * g;
    return Two(fminf(q.lo(), 1e30f), fminf(q.hi(), 1e30f));
  }
  template <bool GELU>
  __device__ __forceinline__ static Two sigmoid(Two g, Two squares) {
    constexpr float kLog2e = 1.4426950408889634f;
    const Two z = GELU ? g * fma(Two(kLog2e * kC3), squares, Two(kLog2e * kC1)) : g * Two(kLog2e);
    // of e = 2^-|z|, which is 1 at most: 1 / (1 + e), or e / (1 + e) where z < 0, small as it may be
    const float e0 = exp2_near(-fabsf(z.lo())), e1 = exp2_near(-fabsf(z.hi()));
    const Two t = Two(e0, e1) + Two(1.f);
    return Two(z.lo() < 0.f ? e0 : 1.f, z.hi() < 0.f ? e1 : 1.f) * Two(reciprocal_near(t.lo()), reciprocal_near(t.hi()));
  }
  // f(g) up
  template <bool GELU>
  __device__ __forceinline__ static Two act(Two g, Two up) {
    return g * sigmoid<GELU>(g, GELU ? square(g) : g) * up;
  }
  // d: gradient of act
  template <bool GELU>
  __device__ __forceinline__ static void grad(Two g, Two up, Two d, Two* d_gate, Two* d_up, Two* act) {
    const Two squares = GELU ? square(g) : g;
    const Two s = sigmoid<GELU>(g, squares), f = g * s, rest = fma(s, Two(-1.f), Two(1.f));
    Two slope = f * rest;  // f' = s + f (1 - s) z'
    if (GELU) slope = slope * fma(Two(3.f * kC3), squares, Two(kC1));
    *d_gate = d * up * (slope + s);
    *d_up = d * f;
    *act = f * up;
  }
  // One at a time, where speed does not matter
  __device__ __forceinline__ float act(float g, float up) const {
    return (gelu ? act<true>(Two(g), Two(up)) : act<false>(Two(g), Two(up))).lo();
  }
  __device__ __forceinline__ void grad(float g, float up, float d, float* d_gate, float* d_up, float* of_act) const {
    Two a, b, c;
    if (gelu) grad<true>(Two(g), Two(up), Two(d), &a, &b, &c);
    else grad<false>(Two(g), Two(up), Two(d), &a, &b, &c);
    *d_gate = a.lo();
    *d_up = b.lo();
    *of_act = c.lo();
  }
};

}  // namespace sptir
#endif  // SPARSETIR_B200_GATE_CUH_
