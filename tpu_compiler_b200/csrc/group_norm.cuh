// Group normalisation with an activation, channels last: per image n and group g of c / groups neighbouring channels
//   mean = E[x], var = E[(x - mean)^2] over the image's pixels and the group's channels,
//   y = act((x - mean) / sqrt(var + eps) * gamma[channel] + beta[channel]).
// groups = 1 on a [tokens, channels] tensor is layer norm. Statistics and affine in fp32, one rounding at the end.
#pragma once
#include "activation.cuh"
#include "host_common.h"

namespace tpucb {

struct GroupNormArgs {
  const void *in;
  void *out;
  const float *gamma, *beta; // [cp], zero behind c
  int n, pixels, c, cp, groups, cg;
  float eps;
};

template <typename T> struct NormType;
template <> struct NormType<float> {
  static constexpr bool kF32 = true;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct NormType<uint16_t> {
  static constexpr bool kF32 = false;
  static __device__ __forceinline__ float get(uint16_t v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ uint16_t put(float v) { return (uint16_t)bf16x2_ieee(v, v); }
};

__device__ __forceinline__ float block_sum(float v, float *red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) v += red[i];
  return v;
}

// One block per image and group, three passes over its values.
template <typename T, int ACT> __global__ void group_norm_kernel(GroupNormArgs a) {
  pdl_prologue();
  __shared__ float red[32];
  const int img = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
  const size_t base = (size_t)img * a.pixels * a.cp + (size_t)g * a.cg;
  const T *in = (const T *)a.in + base;
  T *out = (T *)a.out + base;
  const size_t count = (size_t)a.pixels * a.cg;
  auto at = [&](size_t i) { // offset of the group's value i
    const unsigned ch = div_rem(i, (unsigned)a.cg);
    return i * a.cp + ch;
  };
  float s = 0.0f;
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) s += NormType<T>::get(in[at(i)]);
  const float mean = block_sum(s, red) / (float)count;
  s = 0.0f;
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) {
    const float d = NormType<T>::get(in[at(i)]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = rsqrtf(block_sum(s, red) / (float)count + a.eps);
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) {
    const size_t o = at(i);
    const int ch = g * a.cg + (int)(o % a.cp);
    const float v = (NormType<T>::get(in[o]) - mean) * rstd;
    out[o] = NormType<T>::put(activate<ACT, NormType<T>::kF32>(fmaf(v, a.gamma[ch], a.beta[ch])));
  }
}

inline void launch_group_norm(const GroupNormArgs &a, bool f32, int act, cudaStream_t s) {
  with_activation(act, [&](auto k) {
    constexpr int ACT = decltype(k)::value;
    if (f32) launch_k(group_norm_kernel<float, ACT>, (unsigned)(a.n * a.groups), 256, 0, s, a);
    else launch_k(group_norm_kernel<uint16_t, ACT>, (unsigned)(a.n * a.groups), 256, 0, s, a);
  });
}

} // namespace tpucb
