// Inner product with bias, activation and residual: y = act(x W^T + b) + r, for BF16 and fp32 rows.
#pragma once
#include "activation.cuh"
#include "host_common.h"

namespace tpucb {

struct LinearArgs {
  const void *x, *w, *res; // [m][k], [n_pad][k], null or [m][ldy]
  const float *bias;       // [n_pad]
  void *y;                 // [m][ldy]
  int m, k, n, ldy;        // k: with the padding of the channel pitch, whose weights are zero
};

// 64 x 64 results per block of 256 threads, 4 x 4 per thread, fp32 multiply-adds in the order of k.
template <typename T, int ACT> __global__ void __launch_bounds__(256) linear_kernel(LinearArgs a) {
  pdl_prologue();
  constexpr int BK = 16;
  constexpr bool F32 = sizeof(T) == 4;
  __shared__ float xs[BK][65], ws[BK][65];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  auto get = [](const void *p, size_t i) { return F32 ? ((const float *)p)[i] : bf16_bits_to_f32(((const uint16_t *)p)[i]); };
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.k; k0 += BK) {
    for (int i = threadIdx.x; i < 64 * BK; i += 256) {
      const int r = i / BK, k = i % BK;
      xs[k][r] = m0 + r < a.m && k0 + k < a.k ? get(a.x, (size_t)(m0 + r) * a.k + k0 + k) : 0.0f;
      ws[k][r] = n0 + r < a.ldy && k0 + k < a.k ? get(a.w, (size_t)(n0 + r) * a.k + k0 + k) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = m0 + ty * 4 + i;
    if (row >= a.m) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = n0 + tx * 4 + j;
      if (ch >= a.n) break;
      const size_t o = (size_t)row * a.ldy + ch;
      float v = activate<ACT, F32>(both(acc[i][j] + a.bias[ch])).lo();
      if (a.res) v += get(a.res, o);
      if (F32) ((float *)a.y)[o] = v;
      else ((uint16_t *)a.y)[o] = (uint16_t)bf16x2_ieee(v, v);
    }
  }
}

inline void launch_linear(const LinearArgs &a, bool f32, int act, cudaStream_t s) {
  const dim3 grid((a.n + 63) / 64, (a.m + 63) / 64);
  with_activation(act, [&](auto k) {
    constexpr int ACT = decltype(k)::value;
    if (f32) launch_k(linear_kernel<float, ACT>, grid, 256, 0, s, a);
    else launch_k(linear_kernel<uint16_t, ACT>, grid, 256, 0, s, a);
  });
}

} // namespace tpucb
