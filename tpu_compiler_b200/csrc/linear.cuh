// Inner product with bias, activation and residual in fp32: y[m][n] = act(x[m][k] w[n][k]^T + bias) + residual on the multiply-add pipe.
// (Three TF32 products on the tensor cores, as the convolutions have them, lose a factor of 2 to 4 of fp32's precision at these K; calibration,
// whose pass this is, can wait for the exact one.) Bound: 128 multiply-adds per clock and SM, behind the reads of shared memory (60% of their
// slots): 200 x 1024 x 1000 11.8 us with three modules in flight (35 TFLOP/s), 2000 x 1000 x 2000 193 us (41).
//
// A block of 128 threads computes 8 RM rows x 64 channels, a thread RM x 4 of them, 8 rows and 16 channels apart. Both operands lie along K
// in memory and so in shared memory (rows of 16 values and 4 of padding: eight rows' 16 bytes meet no bank twice); packed multiply-adds take
// two K at once, so that a sum is two partial ones, of the even and the odd K. (8 x 8 per thread halve the reads of shared memory, but leave
// two blocks per SM: 209 us instead of 193 at 2000 x 1000 x 2000; 64 rows spill registers.) A cluster of up to eight blocks shares a tile's K and adds up the partial
// sums through shared memory in the order of K. RM is the one whose tiles fit the rows best: 200 rows are five tiles of 40, not four of 64.
#pragma once
#include "activation.cuh"
#include "conv_big.cuh"

namespace tpucb {

struct LinearF32Args {
  const float *x, *w, *res; // [m][k], [n_pad][k], null or [m][ldy]
  const float *bias;        // [n_pad]
  float *y;                 // [m][ldy]
  int m, k, n, n_pad, ldy;  // k, n_pad and ldy with the padding of the channel pitch (multiples of 4), whose weights and bias are zero
  int split, act;
};

constexpr int kF32K = 16, kF32Pitch = kF32K + 4, kF32N = 64, kF32Threads = 128;
// as many stages as 48 KiB hold, eight at most
__host__ __device__ constexpr int linear_f32_stages(int rm) {
  const int fit = 48 * 1024 / ((8 * rm + kF32N) * kF32Pitch * 4);
  return fit > 8 ? 8 : fit;
}
__host__ __device__ constexpr size_t linear_f32_smem(int rm) {
  const size_t ring = (size_t)linear_f32_stages(rm) * (8 * rm + kF32N) * kF32Pitch * 4, sums = (size_t)8 * rm * kF32N * 4;
  return ring > sums ? ring : sums;
}

namespace ptx {
// 16 bytes to shared memory, zeros where there is nothing to read
__device__ __forceinline__ void cp_async16(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
} // namespace ptx

template <int RM> __global__ void __launch_bounds__(kF32Threads, 4) linear_f32_kernel(const LinearF32Args a) {
  extern __shared__ float smem_f32[];
  constexpr int BM = 8 * RM, RN = kF32N / 16, kF32Stages = linear_f32_stages(RM);
  const int rank = (int)ptx::cluster_rank();
  const int n_tiles = (a.n_pad + kF32N - 1) / kF32N, tile = (int)blockIdx.x / a.split, tm = tile / n_tiles;
  const int m0 = tm * BM, n0 = (tile - tm * n_tiles) * kF32N;
  const int blocks = (a.k + kF32K - 1) / kF32K;
  const int kb0 = (int)((long long)rank * blocks / a.split), nk = (int)((long long)(rank + 1) * blocks / a.split) - kb0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ty = (warp >> 1) * 4 + (lane >> 3), tx = (warp & 1) * 8 + (lane & 7);
  const uint32_t base = ptx::smem_u32(smem_f32);
  constexpr uint32_t kStage = (BM + kF32N) * kF32Pitch * 4, kW = BM * kF32Pitch * 4;

  // Rows of four 16-byte pieces: a thread copies the same piece of every 32nd row, of x and of w. Rows behind the last are those of row 0 (their
  // results are not written); K behind the last is zero.
  constexpr int kXCopies = (BM + 31) / 32, kWCopies = kF32N / 32;
  const int piece = threadIdx.x & 3, row = threadIdx.x >> 2, k_left = a.k - kb0 * kF32K - piece * 4;
  const float *from_x[kXCopies], *from_w[kWCopies];
#pragma unroll
  for (int i = 0; i < kXCopies; ++i) from_x[i] = a.x + (size_t)(m0 + row + 32 * i < a.m ? m0 + row + 32 * i : 0) * a.k + kb0 * kF32K + piece * 4;
#pragma unroll
  for (int i = 0; i < kWCopies; ++i) from_w[i] = a.w + (size_t)(n0 + row + 32 * i < a.n_pad ? n0 + row + 32 * i : 0) * a.k + kb0 * kF32K + piece * 4;
  const uint32_t to = base + (uint32_t)(row * kF32Pitch + piece * 4) * 4;
  auto copy_w = [&](int it, uint32_t stage) {
    const bool there = it * kF32K < k_left;
#pragma unroll
    for (int i = 0; i < kWCopies; ++i) ptx::cp_async16(to + stage + kW + (uint32_t)(32 * i * kF32Pitch * 4), there ? from_w[i] + it * kF32K : a.w, there);
  };
  auto copy_x = [&](int it, uint32_t stage) {
    const bool there = it * kF32K < k_left;
#pragma unroll
    for (int i = 0; i < kXCopies; ++i)
      if (BM % 32 == 0 || row + 32 * i < BM)
        ptx::cp_async16(to + stage + (uint32_t)(32 * i * kF32Pitch * 4), there ? from_x[i] + it * kF32K : a.x, there);
  };
  for (int i = 0; i < kF32Stages - 1; ++i)
    if (i < nk) copy_w(i, (uint32_t)i * kStage); // weights are written at load time only: they need not wait for the previous kernel
  pdl_wait();
  pdl_trigger();
  for (int i = 0; i < kF32Stages - 1; ++i) {
    if (i < nk) copy_x(i, (uint32_t)i * kStage);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  Pair acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = both(0.0f);
  uint32_t stage = 0, next = (kF32Stages - 1) * kStage;
  for (int it = 0; it < nk; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kF32Stages - 2) : "memory");
    __syncthreads(); // the block's copies of this stage are there, and the stage that comes next has been read by all
    if (it + kF32Stages - 1 < nk) {
      copy_w(it + kF32Stages - 1, next);
      copy_x(it + kF32Stages - 1, next);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float *xs = smem_f32 + stage / 4 + ty * kF32Pitch, *ws = smem_f32 + (stage + kW) / 4 + tx * kF32Pitch;
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
        for (int j = 0; j < RN; ++j) acc[i][j] = fma(Pair(x[i].x, x[i].y), Pair(w[j].x, w[j].y), acc[i][j]);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = fma(Pair(x[i].z, x[i].w), Pair(w[j].z, w[j].w), acc[i][j]);
    }
    stage = stage == (kF32Stages - 1) * kStage ? 0 : stage + kStage;
    next = next == (kF32Stages - 1) * kStage ? 0 : next + kStage;
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
      // (padded channels stay zero: an infinity of x times their weights is a NaN)
      const int valid = a.n - n0 - col;
      *reinterpret_cast<float4 *>(a.y + o) = make_float4(v0.lo(), valid > 1 ? v0.hi() : 0.0f, valid > 2 ? v1.lo() : 0.0f, valid > 3 ? v1.hi() : 0.0f);
    }
  });
  __syncwarp();
  if (a.split > 1) ptx::cluster_sync(); // the others have read this block's sums
}

inline void launch_linear_f32(const LinearF32Args &a, const LinearF32Plan &p, cudaStream_t s) {
  PdlConvScope conv_class;
  auto go = [&](auto rm) {
    constexpr int RM = decltype(rm)::value;
    static_assert(linear_f32_smem(RM) <= 48 * 1024, "shared memory that a kernel has unasked");
    launch_cluster_k(p.split, linear_f32_kernel<RM>, p.grid, kF32Threads, linear_f32_smem(RM), s, a);
  };
  switch (p.rm) {
  case 1: go(std::integral_constant<int, 1>()); break;
  case 2: go(std::integral_constant<int, 2>()); break;
  case 3: go(std::integral_constant<int, 3>()); break;
  case 4: go(std::integral_constant<int, 4>()); break;
  case 5: go(std::integral_constant<int, 5>()); break;
  case 6: go(std::integral_constant<int, 6>()); break;
  default: go(std::integral_constant<int, 7>());
  }
}

} // namespace tpucb
