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

// Two values in a register pair: the packed instructions round each half as the single ones do and take one issue slot for two.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ float lo() const { return __uint_as_float((uint32_t)v); }
  __device__ __forceinline__ float hi() const { return __uint_as_float((uint32_t)(v >> 32)); }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair both(float v) { return Pair(v, v); }
// two BF16 values of a word
__device__ __forceinline__ Pair pair_of_bf16(uint32_t w) { return Pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// 1 / a of each half with one reciprocal: 1 / lo = hi / (lo hi). The special-function unit (16 results per clock and SM) bounds
// the activations of memory-bound passes: 2 results per value are 30 us for 2^26 values on 148 SMs, 1.5 are 22. |lo hi| must stay in
// range.
__device__ __forceinline__ Pair reciprocals(Pair a) {
  const float r = rcp_approx(a.lo() * a.hi());
  return Pair(a.hi() * r, a.lo() * r);
}
// v / (1 + 2^t). The exponent is held at 62, so that the product of two denominators stays in range, and for large t the quotient goes to zero itself,
// because v may be large (left at its last value SiLU of -1e20 was -87). Minus infinity times that zero is a NaN, as where the definition is computed.
//   fp32: a factor that falls from 1 at t = 60 to 0 at t = 61: what is lost is below 2^-60 |v|.
//   BF16: 2^-61 is taken from the quotient in the multiply-add that forms it, which saturates at zero. Up to t = 52, SiLU of -36, that is less than
//   half a step of the result; in all it is below 2^-61 |v|. (The factor's three instructions: 64 x 256 x 32 x 32 with SiLU 14.7 -> 15.3 us with three
//   modules in flight, these none.)
template <bool F32> __device__ __forceinline__ Pair over_one_plus_exp2(Pair v, Pair t) {
  const Pair d = Pair(ex2_approx(fminf(t.lo(), 62.0f)), ex2_approx(fminf(t.hi(), 62.0f))) + both(1.0f);
  if (F32) return v * Pair(__saturatef(61.0f - t.lo()), __saturatef(61.0f - t.hi())) * reciprocals(d);
  const float r = rcp_approx(d.lo() * d.hi());
  return v * Pair(__saturatef(fmaf(d.hi(), r, -4.3368087e-19f)), __saturatef(fmaf(d.lo(), r, -4.3368087e-19f)));
}

// gelu(v) = v Phi(v) = max(v, 0) - |v| Q(|v|), with the upper tail of the normal distribution Q(a) = erfc(a / sqrt 2) / 2 =
// e^(-a^2/2) P(1 / (1 + p a)): no cancellation on either side. The polynomials P are this file's own minimax fits of
// e^(a^2/2) Q(a) over a in [0, 14] (beyond, Q is below 1e-44): largest relative error 2.4e-5 for BF16 results, a hundredth of
// their rounding, and 3.1e-7 for fp32 ones. The exponent's rounding adds up to 1.5 2^-24 a^2 of the tail: in all 8e-7 of the value
// down to -3, 1.3e-6 to -5 (a value of 1.4e-6), 7.6e-6 to -12 (2e-32), measured. (Beyond 2^40 the reciprocals
// of a pair would leave the range: a is held there.) v / 2 + |v| / 2 is max(v, 0), and for minus infinity a NaN, as where the definition is computed.
template <bool F32> __device__ __forceinline__ Pair gelu_exact(Pair v) {
  const Pair a(fminf(fabsf(v.lo()), 1.0995116e12f), fminf(fabsf(v.hi()), 1.0995116e12f));
  const Pair t = reciprocals(fma(both(0.35f), a, both(1.0f))), x = a * a * both(-0.7213475204444817f);
  const Pair e(ex2_approx(x.lo()), ex2_approx(x.hi()));
  Pair q; // -P
  if (F32) {
    q = fma(both(-0.04894244623667017f), t, both(0.2021192868271973f));
    q = fma(q, t, both(-0.24064081895892164f));
    q = fma(q, t, both(0.01702343620260618f));
    q = fma(q, t, both(-0.15596148733152987f));
    q = fma(q, t, both(-0.13335509625098455f));
    q = fma(q, t, both(-0.14027034361266144f));
    q = fma(q, t, both(2.731554772757582e-05f));
  } else {
    q = fma(both(0.09778110211354195f), t, both(-0.278881467362648f));
    q = fma(q, t, both(-0.010946683641198824f));
    q = fma(q, t, both(-0.17298857188677733f));
    q = fma(q, t, both(-0.13469103084119843f));
    q = fma(q, t, both(-0.0002850549969567228f));
  }
  const Pair h = v * both(0.5f);
  return fma(a, q * e, Pair(h.lo() + fabsf(h.lo()), h.hi() + fabsf(h.hi())));
}
template <int ACT, bool F32> __device__ __forceinline__ Pair activate(Pair v) {
  if (ACT == ACT_RELU) return Pair(v.lo() < 0.0f ? 0.0f : v.lo(), v.hi() < 0.0f ? 0.0f : v.hi());
  if (ACT == ACT_SILU) return over_one_plus_exp2<F32>(v, v * both(-1.4426950408889634f));
  if (ACT == ACT_GELU) return gelu_exact<F32>(v);
  // 0.5 v (1 + tanh u) = v / (1 + e^(-2u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
  if (ACT == ACT_GELU_TANH) return over_one_plus_exp2<F32>(v, v * fma(v * v, both(-0.10294324f), both(-2.3022082f)));
  return v;
}
// `use` is called with the activation as a compile-time constant, in a kernel or on the host
#pragma nv_exec_check_disable
template <class Use> __host__ __device__ inline void with_activation(int act, Use use) {
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
