// Inner product with bias, activation and residual on the tensor cores: y[m][n] = act(x[m][k] w[n][k]^T + bias) + residual, BF16
// operands, fp32 accumulators in tensor memory, one rounding.
//
// Rows of x lie on the lanes of tensor memory, rows of w (channels) on its columns: an epilogue thread owns a row, whose residual it reads in
// whole 32-byte sectors.
//
// linear_pair_kernel, for launches of many tiles: a persistent pair of CTAs (two SMs, tcgen05 cta_group::2) computes tiles of 256
//   rows x nt channels; each CTA holds 128 of the rows and half of the channels' weights, so that a K block of 64 costs an SM
//   (128 + nt / 2) x 128 bytes of copies. Accumulators are double-buffered: the epilogue of a tile runs beside the next one's loop; its
//   warps write 32 rows x 32 channels through shared memory by bulk tensor stores, clipped by their map (sectors stored by the threads:
//   8192 x 256 x 8192 59 us, now 47). Bound by the tensor pipe, and with work in flight all the time by the power limit: 8192 x 4096 x 4096
//   with a residual 176 us in a single launch (1.56 PFLOP/s, pipe 92% active), 210 to 229 with three modules in flight. The accumulators cut
//   what an fp32 multiply-add rounds: about 1e-5 of a value at K = 4096, which moves one BF16 result in 400 to its neighbour.
// linear_split_kernel, for the others, down to one row: tiles of 128 rows x nt channels, and a cluster of up to eight CTAs that
//   share a tile's K, so that few rows still draw weights through all SMs. The partial sums meet in shared memory: every CTA adds up
//   its share of the columns from all of the cluster, in the order of K (no atomics, the same bits every time), and finishes it.
//   Copies of x take as many rows as there are; the tensor memory is given back before a CTA waits for the others of its
//   cluster (two clusters on the same SMs could otherwise wait for each other's). Bound by memory where K and the channels are long
//   (1 x 4096 x 4096 with a residual 6.6 us with three modules in flight, 78% of the copy rate; 1 x 8192 x 8192 19.9), by latency below.
// Weights are fetched before the previous kernel's results are waited for (programmatic dependent launch). Every wait is bounded as in
// conv_gemm_i8.cuh.
#pragma once
#include "activation.cuh"
#include "conv_plan.cuh"

namespace tpucb {

// (its sizes: linear_tc_plan)
struct LinearTcParams {
  int m, n, n_pad; // rows; channels, without and with the padding of the pitch, whose weights and bias are zero
  int ldy;        // pitch of y and the residual, in values
  int k_blocks;   // of 64 values
  int nt;         // channels per tile: a multiple of 16 (pair: of 64), at most 256
  int split;      // CTAs that share a tile's K
  int a_rows;     // rows of x per copy
  int stages;
  uint32_t tmem_cols, idesc;
  const float *bias;   // for whole tiles of 256 channels
  const uint16_t *res; // or null
  uint16_t *y;
  int *err;
  int wait_rounds, lose_arrival; // self-test of the bounded waits, as in ConvGemmParams
};

constexpr int kSplitThreads = 192;  // copies, MMAs, four epilogue warps
constexpr int kPairEpilogueWarps = 16;
constexpr int kPairThreads = 32 * (4 + kPairEpilogueWarps); // copies of x, of w, MMAs, one idle

namespace ptx {
__device__ __forceinline__ void ld_global_32b(const void *p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void st_global_32b(void *p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tcgen05_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
      "%29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory"); }
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
} // namespace ptx

// Sixteen channels of one row: bias, activation, residual, rounding. Padded channels become zero whatever is in x: an infinity times their zero
// weights would be a NaN, which the next inner product would add to its sums. (A map that ends with the channels does not keep the bulk stores from
// them: they write 16 bytes at a time.)
template <int ACT> __device__ __forceinline__ void linear_finish16(const uint32_t *acc, const LinearTcParams &p, size_t at, int col, uint32_t (&o)[8]) {
  uint32_t r[8];
  const bool residual = p.res && col < p.n_pad;
  if (residual) ptx::ld_global_32b(p.res + at, r);
  const float4 *bias = reinterpret_cast<const float4 *>(p.bias + col);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float4 b = __ldg(bias + q);
    Pair v[2] = {activate<ACT, false>(Pair(__uint_as_float(acc[4 * q]), __uint_as_float(acc[4 * q + 1])) + Pair(b.x, b.y)),
                 activate<ACT, false>(Pair(__uint_as_float(acc[4 * q + 2]), __uint_as_float(acc[4 * q + 3])) + Pair(b.z, b.w))};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (residual) v[j] = v[j] + pair_of_bf16(r[2 * q + j]);
      o[2 * q + j] = bf16x2_ieee(v[j].lo(), v[j].hi());
    }
  }
  if (col + 16 > p.n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] &= (col + 2 * j < p.n ? 0xffffu : 0u) | (col + 2 * j + 1 < p.n ? 0xffff0000u : 0u);
  }
}
template <int ACT> __device__ __forceinline__ void linear_store16(const uint32_t *acc, const LinearTcParams &p, int row, int col) {
  const size_t at = (size_t)row * p.ldy + col;
  uint32_t o[8];
  linear_finish16<ACT>(acc, p, at, col, o);
  ptx::st_global_32b(p.y + at, o);
}

// A role has given up: no copy may be in flight when the CTA's shared memory is released, and the barriers that would tell may
// count copies that were never started. A copy lands within microseconds, so 2 ms are waited for, by the clock.
__device__ __forceinline__ void drain_copies() {
  unsigned long long t0, t1;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (int i = 0; i < (1 << 20); ++i) {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
    if (t1 - t0 > 2000000ull) break;
    __nanosleep(1000);
  }
}

template <int ACT>
__global__ void __launch_bounds__(kSplitThreads)
linear_split_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const LinearTcParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - raw);
  const uint32_t bar_full = base, bar_empty = base + 128, bar_acc = base + 256;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + 264);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + 268);
  const uint32_t ring = base + kLinearHeader;

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)ptx::cluster_rank();
  const int n_tiles = (p.n_pad + p.nt - 1) / p.nt;
  const int tile = (int)blockIdx.x / p.split, tm = tile / n_tiles, tn = tile - tm * n_tiles;
  const int m0 = tm * 128, n0 = tn * p.nt;
  const int kb0 = (int)((long long)rank * p.k_blocks / p.split), nk = (int)((long long)(rank + 1) * p.k_blocks / p.split) - kb0;
  const uint32_t a_bytes = (uint32_t)p.a_rows * 128u, b_bytes = (uint32_t)p.nt * 128u;
  // (The tensor core reads 128 rows of x whatever the copies bring: what lies behind them gives results of rows that nobody reads.)
  const uint32_t b_at = (a_bytes + 1023u) & ~1023u, stage_bytes = b_at + ((b_bytes + 1023u) & ~1023u);
  const int wait_rounds = p.wait_rounds > 0 ? p.wait_rounds : 1024;

  const int ahead = min(nk, p.stages);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 2); // weights, rows
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    ptx::mbar_init(bar_acc, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    *abort_flag = 0;
    // weights are written at load time only: they need not wait for the previous kernel, nor for the other warps
    for (int i = 0; i < ahead; ++i) {
      ptx::mbar_expect_tx(bar_full + 8 * i, b_bytes);
      ptx::tma_load_2d(ring + (uint32_t)i * stage_bytes + b_at, &tmW, bar_full + 8 * i, (kb0 + i) * 128, n0);
    }
  }
  if (threadIdx.x == 64) asm volatile("prefetch.tensormap [%0];" ::"l"(&tmX) : "memory");
  if (warp == 1) ptx::tcgen05_alloc(ptx::smem_u32(tmem_slot), p.tmem_cols);
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  pdl_trigger(); // (behind the allocation: a successor's CTA on this SM does not take what this one needs)
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;

  if (warp == 0) {
    pdl_wait();
    if (ptx::elect_one()) {
      for (int i = 0; i < ahead; ++i) {
        ptx::mbar_expect_tx(bar_full + 8 * i, a_bytes);
        ptx::tma_load_2d(ring + (uint32_t)i * stage_bytes, &tmX, bar_full + 8 * i, (kb0 + i) * 128, m0);
      }
    }
    __syncwarp();
    int s = 0;
    uint32_t ph = 0;
    for (int i = ahead; i < nk; ++i) {
      if (!ptx::mbar_wait_warp(bar_empty + 8 * s, ph, abort_flag, wait_rounds)) {
        wait_expired(p.err, abort_flag, kErrEmptyWait);
        break;
      }
      if (ptx::elect_one()) {
        const uint32_t at = ring + (uint32_t)s * stage_bytes, fb = bar_full + 8 * s;
        ptx::mbar_expect_tx(fb, b_bytes);
        ptx::tma_load_2d(at + b_at, &tmW, fb, (kb0 + i) * 128, n0);
        ptx::mbar_expect_tx(fb, a_bytes);
        ptx::tma_load_2d(at, &tmX, fb, (kb0 + i) * 128, m0);
      }
      if (++s == p.stages) {
        s = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    const uint64_t desc0 = make_kmajor_desc(ring, 128);
    const uint32_t hi = (uint32_t)(desc0 >> 32), lo0 = (uint32_t)desc0, step = stage_bytes >> 4, w_at = b_at >> 4;
    int s = 0;
    uint32_t ph = 0, lo = lo0;
    for (int i = 0; i < nk; ++i) {
      if (!ptx::mbar_wait_warp(bar_full + 8 * s, ph, abort_flag, wait_rounds)) {
        wait_expired(p.err, abort_flag, kErrFullWait);
        ok = false;
        break;
      }
      ptx::tcgen05_fence_after();
      if (ptx::elect_one()) {
        ptx::tcgen05_mma_i8_kblock<4, 1>(tmem, lo, lo + w_at, hi, p.idesc, i > 0 ? 1u : 0u);
        ptx::tcgen05_commit(bar_empty + 8 * s);
      }
      lo += step;
      if (++s == p.stages) {
        s = 0;
        ph ^= 1u;
        lo = lo0;
      }
    }
    if (ok && !p.lose_arrival && ptx::elect_one()) ptx::tcgen05_commit(bar_acc);
    __syncwarp();
  } else {
    const int cols = min(p.nt, p.n_pad - n0);
    if (lane * 32 < cols) ptx::prefetch_l2(p.bias + n0 + lane * 32);
    pdl_wait(); // the residual
    // a kernel that gave up earlier ends this one's waits
    if (threadIdx.x == 64 && *reinterpret_cast<volatile int *>(p.err) != 0) *abort_flag = 1;
    if (p.res && m0 + (warp & 3) * 32 + lane < p.m)
      for (int c = rank * 64; c < cols; c += p.split * 64) ptx::prefetch_l2(p.res + (size_t)(m0 + (warp & 3) * 32 + lane) * p.ldy + n0 + c);
    ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_acc, 0, abort_flag, wait_rounds));
    if (!ok) wait_expired(p.err, abort_flag, kErrAccWait);
    ptx::tcgen05_fence_after();
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const int rows = min(128, (p.m - m0 + 31) & ~31); // of the partial sums that are exchanged
    if (ok && quarter * 32 < rows) {
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
      for (int c = 0; c < cols; c += 16) {
        uint32_t r[16];
        ptx::tcgen05_ld_x16(acc + (uint32_t)c, r);
        ptx::tcgen05_wait_ld();
        if (p.split == 1) {
          if (m0 + row < p.m) linear_store16<ACT>(r, p, m0 + row, n0 + c);
          __syncwarp();
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) // [column][row]: a warp writes 128 bytes in a row; the copies that were here have been consumed
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring + 4u * (uint32_t)((c + j) * rows + row)), "r"(r[j]) : "memory");
        }
      }
    }
  }

  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) drain_copies();
    ptx::tcgen05_fence_after();
    ptx::tcgen05_dealloc(tmem, p.tmem_cols);
  }
  if (p.split > 1) {
    ptx::cluster_sync();
    const int rows = min(128, (p.m - m0 + 31) & ~31);
    const int chunks = (min(p.nt, p.n_pad - n0) + 15) / 16, mine = (chunks - rank + p.split - 1) / p.split;
    if (*abort_flag == 0) {
      for (int i = threadIdx.x; i < rows * mine; i += kSplitThreads) {
        const int row = i % rows, c = (rank + i / rows * p.split) * 16;
        if (m0 + row >= p.m) continue;
        float acc[16] = {};
        for (int s = 0; s < p.split; ++s) {
          const uint32_t from = ptx::map_cluster(ring + 4u * (uint32_t)(c * rows + row), (uint32_t)s);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[j] += ptx::ld_cluster_f32(from + 4u * (uint32_t)(j * rows));
        }
        linear_store16<ACT>(reinterpret_cast<const uint32_t *>(acc), p, m0 + row, n0 + c);
      }
    }
    __syncwarp();
    ptx::cluster_sync(); // the others have read this CTA's sums
  }
}

template <int ACT>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
                   const LinearTcParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - raw);
  const uint32_t bar_full = base, bar_empty = base + 128, bar_acc_full = base + 256, bar_acc_empty = base + 272;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + 288);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + 292);
  const uint32_t ring = base + kLinearHeader + kPairStaging;

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_rank();
  const int n_tiles = (p.n_pad + p.nt - 1) / p.nt, m_tiles = (p.m + 255) / 256, total = n_tiles * m_tiles;
  const int first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;
  const uint32_t a_bytes = 128u * 128u, b_bytes = (uint32_t)(p.nt / 2) * 128u, stage_bytes = a_bytes + b_bytes;
  const int wait_rounds = p.wait_rounds > 0 ? p.wait_rounds : 1024;

  if (threadIdx.x == 0) {
    const int gave_up = *reinterpret_cast<volatile int *>(p.err);
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 2); // one arrival per copying warp, with the bytes of both CTAs
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(bar_acc_full + 8 * b, 1);
      ptx::mbar_init(bar_acc_empty + 8 * b, 2 * kPairEpilogueWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = gave_up; // (the CTAs of a pair may see different values: both go on, within their bounded waits)
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(ptx::smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  ptx::tcgen05_fence_after();
  pdl_trigger();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t lead_full = ptx::map_cluster(bar_full, 0); // barriers of the first CTA, which counts both's copies and issues the MMAs

  if (warp <= 1) {
    const bool rows = warp == 0;
    if (rows) pdl_wait(); // weights are written at load time only
    const uint32_t bytes = rows ? a_bytes : b_bytes, dst0 = ring + (rows ? 0u : a_bytes);
    const CUtensorMap *map = rows ? &tmX : &tmW;
    int it = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += step) {
      const int tm = tile / n_tiles, tn = tile - tm * n_tiles;
      const int y = rows ? tm * 256 + (int)rank * 128 : tn * p.nt + (int)rank * (p.nt / 2);
      for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
        if (it >= p.stages && !ptx::mbar_wait_warp(bar_empty + 8 * s, ph ^ 1u, abort_flag, wait_rounds)) {
          wait_expired(p.err, abort_flag, kErrEmptyWait);
          ok = false;
          break;
        }
        if (ptx::elect_one()) {
          if (rank == 0) ptx::mbar_expect_tx(bar_full + 8 * s, 2 * bytes);
          ptx::big_load_2d<2>(dst0 + (uint32_t)s * stage_bytes, map, lead_full + 8 * s, kb * 128, y);
        }
        if (++s == p.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
    if (!ok || *abort_flag) drain_copies();
  } else if (warp == 2) {
    if (rank == 0) {
      const uint64_t desc0 = make_kmajor_desc(ring, 128);
      const uint32_t hi = (uint32_t)(desc0 >> 32), lo0 = (uint32_t)desc0, stage_step = stage_bytes >> 4, w_at = a_bytes >> 4;
      int t = 0, s = 0;
      uint32_t ph = 0, lo = lo0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += step, ++t) {
        const int buf = t & 1;
        if (t >= 2) {
          if (!ptx::mbar_wait_warp(bar_acc_empty + 8 * buf, (uint32_t)(((t >> 1) - 1) & 1), abort_flag, wait_rounds)) {
            wait_expired(p.err, abort_flag, kErrAccWait);
            break;
          }
          ptx::tcgen05_fence_after();
        }
        const uint32_t d = tmem + (uint32_t)buf * 256u;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!ptx::mbar_wait_warp(bar_full + 8 * s, ph, abort_flag, wait_rounds)) {
            wait_expired(p.err, abort_flag, kErrFullWait);
            ok = false;
            break;
          }
          ptx::tcgen05_fence_after();
          if (ptx::elect_one()) {
            ptx::big_mma<2, 1>(d, lo, lo + w_at, hi, p.idesc, kb > 0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < 4; ++k) ptx::big_mma<2, 1>(d, lo + 2 * k, lo + w_at + 2 * k, hi, p.idesc, 1u);
            ptx::big_commit<2>(bar_empty + 8 * s);
          }
          lo += stage_step;
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
            lo = lo0;
          }
        }
        if (ok && ptx::elect_one()) ptx::big_commit<2>(bar_acc_full + 8 * buf);
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2, row = quarter * 32 + lane;
    const uint32_t lead_acc_empty = ptx::map_cluster(bar_acc_empty, 0), out = base + kLinearHeader + (uint32_t)(warp - 4) * 2048u;
    pdl_wait(); // the residual
    int t = 0;
    for (int tile = first; tile < total; tile += step, ++t) {
      const int tm = tile / n_tiles, tn = tile - tm * n_tiles, buf = t & 1;
      const int m0 = tm * 256 + (int)rank * 128, n0 = tn * p.nt;
      bool ok = *abort_flag == 0;
      if (ok) ok = ptx::mbar_wait_bounded(bar_acc_full + 8 * buf, (uint32_t)((t >> 1) & 1), abort_flag, wait_rounds);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        wait_expired(p.err, abort_flag, kErrAccWait);
        break;
      }
      ptx::tcgen05_fence_after();
      if (m0 + quarter * 32 < p.m) {
        const uint32_t acc = tmem + (uint32_t)buf * 256u + ((uint32_t)(quarter * 32) << 16);
        const int cols = min(p.nt, p.n_pad - n0);
        const bool mine = m0 + row < p.m;
        for (int c = part * 32; c < cols; c += 128) {
          uint32_t r[32];
          ptx::tcgen05_ld_x32(acc + (uint32_t)c, r);
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); // the last store has read the buffer
          ptx::tcgen05_wait_ld();
          __syncwarp();
          if (mine) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t o[8];
              // (columns behind the pitch are clipped by the map; there is bias for them, and no residual)
              linear_finish16<ACT>(r + 16 * q, p, (size_t)(m0 + row) * p.ldy + n0 + c + 16 * q, n0 + c + 16 * q, o);
              // the map's 64-byte swizzle: a row's piece i of 16 bytes lies at i ^ (row / 2 % 4)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + (uint32_t)lane * 64u + (uint32_t)(((2 * q + j) ^ ((lane >> 1) & 3)) << 4)),
                             "r"(o[4 * j]), "r"(o[4 * j + 1]), "r"(o[4 * j + 2]), "r"(o[4 * j + 3]) : "memory");
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            ptx::tma_store_2d(&tmY, out, 2 * (n0 + c), m0 + quarter * 32);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
      ptx::tcgen05_fence_before();
      __syncwarp();
      if (lane == 0 && !p.lose_arrival)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_acc_empty + 8 * buf) : "memory");
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync(); // no CTA leaves while the other's arrivals or operand reads may come to it
  if (warp == 2) {
    ptx::tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

struct LinearTc {
  CUtensorMap tmX, tmW, tmY;
  LinearTcParams p;
  LinearTcPlan plan;
};
template <class Use> inline void with_linear_kernel(const LinearTc &l, int act, Use use) {
  with_activation(act, [&](auto k) {
    constexpr int ACT = decltype(k)::value;
    if (l.plan.pair) use(KernelConstant<linear_pair_kernel<ACT>>());
    else use(KernelConstant<linear_split_kernel<ACT>>());
  });
}
// To be called at load, on the device that will run it (conv_kernel_ready).
inline void linear_kernel_ready(const LinearTc &l, int act) {
  int device = 0;
  TPUCB_CUDA(cudaGetDevice(&device));
  with_linear_kernel(l, act, [&](auto k) {
    static OncePerDevice ready; // one of each kernel
    ready.run(device, [] { TPUCB_CUDA(cudaFuncSetAttribute(decltype(k)::value, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)); });
  });
}
inline void launch_linear_tc(const LinearTc &l, int act, cudaStream_t stream) {
  PdlConvScope conv_class;
  with_linear_kernel(l, act, [&](auto k) {
    constexpr auto kernel = decltype(k)::value;
    if constexpr (std::is_invocable_v<decltype(kernel), CUtensorMap, CUtensorMap, CUtensorMap, LinearTcParams>)
      launch_k(kernel, l.plan.grid, kPairThreads, l.plan.smem, stream, l.tmX, l.tmW, l.tmY, l.p);
    else
      launch_cluster_k(l.plan.split, kernel, l.plan.grid, kSplitThreads, l.plan.smem, stream, l.tmX, l.tmW, l.p);
  });
}

} // namespace tpucb
