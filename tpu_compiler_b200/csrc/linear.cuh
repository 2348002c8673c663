// Inner product with bias, activation and residual in fp32: y[m][n] = act(x[m][k] w[n][k]^T + bias) + residual on the multiply-add pipe.
// (Three TF32 products on the tensor cores, as the convolutions have them, lose a factor of 2 to 4 of fp32's precision at these K; calibration,
// whose pass this is, can wait for the exact one.) Bound: 128 multiply-adds per clock and SM.
//
// A block of 128 threads computes 8 RM rows x 16 RN channels, a thread RM x RN of them, 8 rows and 16 channels apart. Both operands lie along
// K in memory and so in shared memory (rows of 16 values and 4 of padding: eight rows' 16 bytes meet no bank twice); packed multiply-adds
// take two K at once, so that a sum is two partial ones, of the even and the odd K. Per four K a warp's multiply-adds take 4 RM RN clocks
// of its quarter of the SM, and its RM + RN reads of 16 bytes per lane 4 clocks each of the whole SM: 8 x 8 balances the two, smaller ones are
// bound by the reads. A cluster of up to eight blocks shares a tile's K and adds up the partial sums through shared memory in the order
// of K. RM is the one whose tiles fit the rows best: 200 rows are five tiles of 40, not four of 64.
#pragma once
#include "activation.cuh"
#include "conv_big.cuh"

namespace tpucb {

struct LinearF32Args {
  const float *x, *w, *res; // [m][k], [n_pad][k], null or [m][ldy]
  const float *bias;        // [n_pad]
  float *y;                 // [m][ldy]
  int m, k, n_pad, ldy;     // k and ldy with the padding of the channel pitch (multiples of 4), whose weights and bias are zero
  int split, act;
};

constexpr int kF32K = 16, kF32Pitch = kF32K + 4, kF32Threads = 128;
// as many stages as 48 KiB hold, eight at most
__host__ __device__ constexpr int linear_f32_stages(int rm, int rn) {
  const int fit = 48 * 1024 / ((8 * rm + 16 * rn) * kF32Pitch * 4);
  return fit > 8 ? 8 : fit;
}
__host__ __device__ constexpr size_t linear_f32_smem(int rm, int rn) {
  const size_t ring = (size_t)linear_f32_stages(rm, rn) * (8 * rm + 16 * rn) * kF32Pitch * 4, sums = (size_t)8 * rm * 16 * rn * 4;
  return ring > sums ? ring : sums;
}

namespace ptx {
// 16 bytes to shared memory, zeros where there is nothing to read
__device__ __forceinline__ void cp_async16(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
} // namespace ptx

template <int RM, int RN> __global__ void __launch_bounds__(kF32Threads) linear_f32_kernel(const LinearF32Args a) {
  extern __shared__ float smem_f32[];
  constexpr int BM = 8 * RM, kF32N = 16 * RN, kF32Stages = linear_f32_stages(RM, RN);
  const int rank = (int)ptx::cluster_rank();
  const int n_tiles = (a.n_pad + kF32N - 1) / kF32N, tile = (int)blockIdx.x / a.split, tm = tile / n_tiles;
  const int m0 = tm * BM, n0 = (tile - tm * n_tiles) * kF32N;
  const int blocks = (a.k + kF32K - 1) / kF32K;
  const int kb0 = (int)((long long)rank * blocks / a.split), nk = (int)((long long)(rank + 1) * blocks / a.split) - kb0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ty = (warp >> 1) * 4 + (lane >> 3), tx = (warp & 1) * 8 + (lane & 7);
  const uint32_t base = ptx::smem_u32(smem_f32);
  constexpr uint32_t kStage = (BM + kF32N) * kF32Pitch * 4, kW = BM * kF32Pitch * 4;

  // rows of four 16-byte pieces
  auto copy = [&](const float *src, int rows, int row0, int limit, uint32_t to, int kb) {
    for (int i = threadIdx.x; i < rows * 4; i += kF32Threads) {
      const int r = i >> 2, c = kb * kF32K + (i & 3) * 4;
      const bool there = row0 + r < limit && c < a.k;
      ptx::cp_async16(to + (uint32_t)(r * kF32Pitch + (i & 3) * 4) * 4, there ? src + (size_t)(row0 + r) * a.k + c : src, there);
    }
  };
  auto copy_w = [&](int i) { copy(a.w, kF32N, n0, a.n_pad, base + (uint32_t)(i % kF32Stages) * kStage + kW, kb0 + i); };
  auto copy_x = [&](int i) { copy(a.x, BM, m0, a.m, base + (uint32_t)(i % kF32Stages) * kStage, kb0 + i); };
  for (int i = 0; i < kF32Stages - 1; ++i)
    if (i < nk) copy_w(i); // weights are written at load time only: they need not wait for the previous kernel
  pdl_wait();
  pdl_trigger();
  for (int i = 0; i < kF32Stages - 1; ++i) {
    if (i < nk) copy_x(i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  Pair acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = both(0.0f);
  for (int it = 0; it < nk; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kF32Stages - 2) : "memory");
    __syncthreads(); // the block's copies of this stage are there, and the stage that comes next has been read by all
    if (it + kF32Stages - 1 < nk) {
      copy_w(it + kF32Stages - 1);
      copy_x(it + kF32Stages - 1);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float *xs = smem_f32 + (it % kF32Stages) * (kStage / 4) + ty * kF32Pitch, *ws = smem_f32 + (it % kF32Stages) * (kStage / 4) + kW / 4 + tx * kF32Pitch;
#pragma unroll
    for (int k = 0; k < kF32K; k += 4) {
      float4 x[RM], w[RN];
#pragma unroll
      for (int i = 0; i < RM; ++i) x[i] = *reinterpret_cast<const float4 *>(xs + i * 8 * kF32Pitch + k);
#pragma unroll
      for (int j = 0; j < RN; ++j) w[j] = *reinterpret_cast<const float4 *>(ws + j * 16 * kF32Pitch + k);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) {
          acc[i][j] = fma(Pair(x[i].x, x[i].y), Pair(w[j].x, w[j].y), acc[i][j]);
          acc[i][j] = fma(Pair(x[i].z, x[i].w), Pair(w[j].z, w[j].w), acc[i][j]);
        }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) smem_f32[(ty + 8 * i) * kF32N + tx + 16 * j] = acc[i][j].lo() + acc[i][j].hi();
  if (a.split > 1) ptx::cluster_sync();
  else __syncthreads();
  with_activation(a.act, [&](auto act) {
    for (int i = rank * kF32Threads + threadIdx.x; i < BM * (kF32N / 4); i += a.split * kF32Threads) {
      const int row = i / (kF32N / 4), col = i % (kF32N / 4) * 4;
      if (m0 + row >= a.m || n0 + col >= a.n_pad) continue;
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const uint32_t at = base + (uint32_t)(row * kF32N + col) * 4;
      for (int r = 0; r < a.split; ++r) {
        float4 o;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w)
                     : "r"(a.split > 1 ? ptx::map_cluster(at, (uint32_t)r) : at) : "memory");
        s.x += o.x;
        s.y += o.y;
        s.z += o.z;
        s.w += o.w;
      }
      const float4 b = __ldg(reinterpret_cast<const float4 *>(a.bias + n0 + col));
      Pair v0 = activate<decltype(act)::value, true>(Pair(s.x, s.y) + Pair(b.x, b.y));
      Pair v1 = activate<decltype(act)::value, true>(Pair(s.z, s.w) + Pair(b.z, b.w));
      const size_t o = (size_t)(m0 + row) * a.ldy + n0 + col;
      if (a.res) {
        const float4 r = *reinterpret_cast<const float4 *>(a.res + o);
        v0 = v0 + Pair(r.x, r.y);
        v1 = v1 + Pair(r.z, r.w);
      }
      *reinterpret_cast<float4 *>(a.y + o) = make_float4(v0.lo(), v0.hi(), v1.lo(), v1.hi());
    }
  });
  __syncwarp();
  if (a.split > 1) ptx::cluster_sync(); // the others have read this block's sums
}

inline void launch_linear_f32(const LinearF32Args &a, const LinearF32Plan &p, cudaStream_t s) {
  PdlConvScope conv_class;
  auto go = [&](auto rm, auto rn) {
    constexpr int RM = decltype(rm)::value, RN = decltype(rn)::value;
    static_assert(linear_f32_smem(RM, RN) <= 48 * 1024, "shared memory that a kernel has unasked");
    launch_cluster_k(p.split, linear_f32_kernel<RM, RN>, p.grid, kF32Threads, linear_f32_smem(RM, RN), s, a);
  };
  std::integral_constant<int, 4> four;
  switch (p.rm + 8 * (p.rn == 8)) {
  case 1: go(std::integral_constant<int, 1>(), four); break;
  case 2: go(std::integral_constant<int, 2>(), four); break;
  case 3: go(std::integral_constant<int, 3>(), four); break;
  case 4: go(std::integral_constant<int, 4>(), four); break;
  case 5: go(std::integral_constant<int, 5>(), four); break;
  case 6: go(std::integral_constant<int, 6>(), four); break;
  case 7: go(std::integral_constant<int, 7>(), four); break;
  case 8: go(std::integral_constant<int, 8>(), four); break;
  default: go(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  }
}

} // namespace tpucb
