// The activations that group_norm and fully_connected apply in the pass that forms their results, in fp32.
#pragma once
#include "common.cuh"
#include "norm_linear.h"
#include <type_traits>

namespace tpucb {

#ifdef __CUDACC__
// {bf16(hi), bf16(lo)}, rounded to nearest even as IEEE 754 has it: infinities and NaN stay what they are. (The BF16 ops that restate
// the reference turn both into the largest finite value, or a NaN into zero, bf16x2_round_bits; these have nothing to restate.)
__device__ __forceinline__ uint32_t bf16x2_ieee(float lo, float hi) {
  uint32_t p;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
  return p;
}
__device__ __forceinline__ float ex2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// v / (1 + e^-s): an overflowing exponential gives a quotient of zero, as it should
__device__ __forceinline__ float times_sigmoid(float v, float s) { return v * rcp_approx(1.0f + ex2_approx(s * -1.4426950408889634f)); }

// gelu(v) = v Phi(v) = max(v, 0) - |v| Q(|v|), with the upper tail of the normal distribution Q(a) = erfc(a / sqrt 2) / 2 =
// e^(-a^2/2) P(1 / (1 + p a)): no cancellation on either side. The polynomials P are this file's own minimax fits of
// e^(a^2/2) Q(a) over a in [0, 14] (beyond, Q is below 1e-44): largest relative error 2.4e-5 for BF16 results, a hundredth of
// their rounding, and 3.1e-7 for fp32 ones.
template <bool F32> __device__ __forceinline__ float gelu_exact(float v) {
  const float a = fabsf(v), t = rcp_approx(fmaf(0.35f, a, 1.0f)), e = ex2_approx(a * a * -0.7213475204444817f);
  float q;
  if (F32) {
    q = 0.04894244623667017f;
    q = fmaf(q, t, -0.2021192868271973f);
    q = fmaf(q, t, 0.24064081895892164f);
    q = fmaf(q, t, -0.01702343620260618f);
    q = fmaf(q, t, 0.15596148733152987f);
    q = fmaf(q, t, 0.13335509625098455f);
    q = fmaf(q, t, 0.14027034361266144f);
    q = fmaf(q, t, -2.731554772757582e-05f);
  } else {
    q = -0.09778110211354195f;
    q = fmaf(q, t, 0.278881467362648f);
    q = fmaf(q, t, 0.010946683641198824f);
    q = fmaf(q, t, 0.17298857188677733f);
    q = fmaf(q, t, 0.13469103084119843f);
    q = fmaf(q, t, 0.0002850549969567228f);
  }
  return fmaxf(v, 0.0f) - a * (q * e);
}
template <int ACT, bool F32> __device__ __forceinline__ float activate(float v) {
  if (ACT == ACT_RELU) return v < 0.0f ? 0.0f : v;
  if (ACT == ACT_SILU) return times_sigmoid(v, v);
  if (ACT == ACT_GELU) return gelu_exact<F32>(v);
  // 0.5 v (1 + tanh u) = v / (1 + e^(-2u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
  if (ACT == ACT_GELU_TANH) return times_sigmoid(v, v * fmaf(0.07135481627159882f, v * v, 1.5957691216057308f));
  return v;
}
// `use` is called with the activation as a compile-time constant
template <class Use> inline void with_activation(int act, Use use) {
  switch (act) {
  case ACT_RELU: use(std::integral_constant<int, ACT_RELU>()); break;
  case ACT_SILU: use(std::integral_constant<int, ACT_SILU>()); break;
  case ACT_GELU: use(std::integral_constant<int, ACT_GELU>()); break;
  case ACT_GELU_TANH: use(std::integral_constant<int, ACT_GELU_TANH>()); break;
  default: use(std::integral_constant<int, ACT_NONE>());
  }
}
#endif

} // namespace tpucb
