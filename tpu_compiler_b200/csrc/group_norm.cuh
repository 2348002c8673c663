// Group normalisation with an activation, channels last: per image n and group g of c / groups neighbouring channels
//   mean = E[x], var = E[(x - mean)^2] over the image's pixels and the group's channels,
//   y = act((x - mean) / sqrt(var + eps) * gamma[channel] + beta[channel]).
// groups = 1 on a [tokens, channels] tensor is layer norm. Statistics and affine in fp32, one rounding at the end. Bound: memory,
// x read and y written once.
//
// Four forms (group_norm_plan), threads moving vectors of 16 bytes:
//   rows     one pixel per image: a group is contiguous; a warp or a block keeps it in registers;
//   slab     the pixels of an image x a few groups ("chunk") are kept in the registers of a cluster of up to eight blocks, which
//            exchange their statistics through shared memory: x is read once;
//   streamed larger ones: a pass for the statistics, whose last block per chunk joins the partial ones, and a pass that forms
//            the results, in the opposite order, so that it begins with what the L2 still holds;
//   strided  what fits no whole vectors: a block per group, three passes.
// Variances are never differences of large sums: rows and slab take the mean first and then the squares of the distances from it, out of
// the registers; streamed sums distances from the first value that a thread sees of a channel (the error is then at most the
// thread's count times 2^-24 of the variance, even where that value is an outlier: it is part of the variance). Partial ones are joined as
//   M2 = sum M2_i + sum n_i (mean_i - mean)^2.
#pragma once
#include "activation.cuh"
#include "conv_big.cuh"

namespace tpucb {

struct GroupNormArgs {
  const void *in;
  void *out;
  const float *gamma, *beta; // [cp], zero behind c
  int n, pixels, c, cp, groups, cg;
  float eps;
  int act;
  // slab and streamed: chunks of `vecs` vectors = whole groups (the last may have fewer), `parts` blocks share an image's pixels
  int vecs, chunk_groups, chunks, parts, part_pixels;
  float2 *partial;    // streamed: [n][groups][parts] mean, M2
  float2 *stats;      // streamed: [n][groups] mean, 1 / sqrt(var + eps)
  unsigned *arrived;  // streamed: [n][chunks], zero between launches
};

// Sixteen bytes of values
template <typename T> struct NormVec;
template <> struct NormVec<float> {
  static constexpr int N = 4;
  static constexpr bool kF32 = true;
  static __device__ __forceinline__ void get(const uint4 &r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x);
    v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z);
    v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float back(float v) { return v; }
};
template <> struct NormVec<uint16_t> {
  static constexpr int N = 8;
  static constexpr bool kF32 = false;
  static __device__ __forceinline__ void get(const uint4 &r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&v)[8]) {
    return make_uint4(bf16x2_ieee(v[0], v[1]), bf16x2_ieee(v[2], v[3]), bf16x2_ieee(v[4], v[5]), bf16x2_ieee(v[6], v[7]));
  }
  static __device__ __forceinline__ float one(uint16_t v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ uint16_t back(float v) { return (uint16_t)bf16x2_ieee(v, v); }
};

// the activation of a vector's values; which one is the same for the whole launch
template <bool F32, int N> __device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
  switch (act) {
  case ACT_RELU:
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<ACT_RELU, F32>(v[j]);
    break;
  case ACT_SILU:
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<ACT_SILU, F32>(v[j]);
    break;
  case ACT_GELU:
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<ACT_GELU, F32>(v[j]);
    break;
  case ACT_GELU_TANH:
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<ACT_GELU_TANH, F32>(v[j]);
    break;
  default: break;
  }
}
template <int N> __device__ __forceinline__ void load_floats(const float *p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const float4 f = __ldg(reinterpret_cast<const float4 *>(p) + i);
    v[4 * i] = f.x;
    v[4 * i + 1] = f.y;
    v[4 * i + 2] = f.z;
    v[4 * i + 3] = f.w;
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// the sum over the block, in every thread; `red` holds 32 floats and is free again after the next barrier
__device__ __forceinline__ float block_sum(float v, float *red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.0f;
  return warp_sum(v);
}

// ---- rows: groups of one pixel. BLOCK: a block per group, else a warp. NV: vectors per thread.
template <typename T, int NV, bool BLOCK> __global__ void __launch_bounds__(BLOCK ? 1024 : 128) group_norm_rows_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  __shared__ float red[32];
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31, lanes = BLOCK ? blockDim.x : 32;
  const int row = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_prologue();
  if (!BLOCK && row >= a.n * a.groups) return;
  const int img = row / a.groups, g = row - img * a.groups, nvec = (a.cg + V::N - 1) / V::N;
  const size_t base = (size_t)img * a.cp + (size_t)g * a.cg;
  const uint4 *in = reinterpret_cast<const uint4 *>((const T *)a.in + base);
  uint4 *out = reinterpret_cast<uint4 *>((T *)a.out + base);
  uint4 raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = lane + k * lanes;
    raw[k] = i < nvec ? in[i] : make_uint4(0u, 0u, 0u, 0u);
  }
  // (with one group the last vector may end in padded channels)
  auto count = [&](int i) { return min(V::N, a.cg - i * V::N); };
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float x[V::N];
    V::get(raw[k], x);
    const int valid = count(lane + k * lanes);
#pragma unroll
    for (int j = 0; j < V::N; ++j) s += j < valid ? x[j] : 0.0f;
  }
  s = BLOCK ? block_sum(s, red) : warp_sum(s);
  const float mean = s / (float)a.cg;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float x[V::N];
    V::get(raw[k], x);
    const int valid = count(lane + k * lanes);
#pragma unroll
    for (int j = 0; j < V::N; ++j) {
      const float d = j < valid ? x[j] - mean : 0.0f;
      s = fmaf(d, d, s);
    }
  }
  s = BLOCK ? block_sum(s, red) : warp_sum(s);
  const float rstd = rsqrtf(s / (float)a.cg + a.eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = lane + k * lanes;
    if (i >= nvec) continue;
    float x[V::N], ga[V::N], be[V::N];
    load_floats(a.gamma + g * a.cg + i * V::N, ga);
    load_floats(a.beta + g * a.cg + i * V::N, be);
    V::get(raw[k], x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) x[j] = fmaf((x[j] - mean) * rstd, ga[j], be[j]);
    activate_all<V::kF32>(a.act, x);
    const int valid = count(i);
#pragma unroll
    for (int j = 0; j < V::N; ++j) x[j] = j < valid ? x[j] : 0.0f;
    out[i] = V::put(x);
  }
}

// ---- what slab and streamed share: a block of kNormThreads takes pixels x a chunk; a thread keeps to one vector column
constexpr int kNormThreads = 256;
template <typename T> struct NormTile {
  int img, chunk, part, first_group, n_groups; // groups of this chunk
  int px0, px1;                                // this block's pixels
  int v, p, lanes, ch;                         // the thread's vector column, pixel lane, pixel lanes of the block, first channel
  bool active;
  __device__ __forceinline__ NormTile(const GroupNormArgs &a, unsigned block) {
    part = block % a.parts;
    chunk = (block / a.parts) % a.chunks;
    img = block / a.parts / a.chunks;
    first_group = chunk * a.chunk_groups;
    n_groups = min(a.chunk_groups, a.groups - first_group);
    px0 = part * a.part_pixels;
    px1 = min(px0 + a.part_pixels, a.pixels);
    lanes = kNormThreads / a.vecs;
    p = threadIdx.x / a.vecs;
    v = threadIdx.x - p * a.vecs;
    ch = (chunk * a.vecs + v) * NormVec<T>::N;
    active = p < lanes && ch < a.c;
  }
  __device__ __forceinline__ size_t offset(const GroupNormArgs &a, int px) const { return ((size_t)img * a.pixels + px) * a.cp + ch; }
};
// Sums over a chunk's groups of what each thread holds per channel (or, where vectors lie within groups, in all): tab[pixel lane][channel of the
// chunk], a warp per group. `done(group of the chunk, sum)` in lane 0 of that warp.
template <int PER, class Done>
__device__ __forceinline__ void group_sums(const float *tab, int vecs, int lanes, int group_width, int n_groups, Done done) {
  const int width = vecs * PER;
  for (int g = threadIdx.x >> 5; g < n_groups; g += kNormThreads / 32) {
    float s = 0.0f;
    const int total = group_width * lanes;
    for (int e = threadIdx.x & 31; e < total; e += 32) {
      const int p = e / group_width;
      s += tab[p * width + g * group_width + (e - p * group_width)];
    }
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) done(g, s);
  }
}

// ---- slab. ALIGNED: a vector's channels belong to one group. NV: vectors per thread.
template <typename T, bool ALIGNED, int NV> __global__ void __launch_bounds__(kNormThreads) group_norm_slab_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  constexpr int PER = ALIGNED ? 1 : V::N;
  extern __shared__ float smem[];
  float *tab = smem;                                                       // [threads][PER]
  float2 *own = reinterpret_cast<float2 *>(smem + kNormThreads * PER);     // [groups of the chunk]: this block's mean and M2
  float2 *all = own + a.chunk_groups;                                      // mean and 1 / sqrt(var + eps) of the image
  const NormTile<T> t(a, blockIdx.x);
  float ga[V::N], be[V::N];
  int grp[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) grp[j] = min((t.ch + j) / a.cg - t.first_group, t.n_groups - 1); // (padded channels: any group)
  if (t.active) {
    load_floats(a.gamma + t.ch, ga);
    load_floats(a.beta + t.ch, be);
  }
  pdl_prologue();
  const T *in = (const T *)a.in;
  uint4 raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int px = t.px0 + t.p + k * t.lanes;
    if (t.active && px < t.px1) raw[k] = *reinterpret_cast<const uint4 *>(in + t.offset(a, px));
  }
  const int group_width = ALIGNED ? a.cg / V::N : a.cg;
  const float count = (float)(t.px1 - t.px0) * (float)a.cg;
  float acc[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (!(t.active && t.px0 + t.p + k * t.lanes < t.px1)) continue;
    float x[V::N];
    V::get(raw[k], x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) acc[ALIGNED ? 0 : j] += x[j];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) tab[threadIdx.x * PER + j] = acc[j];
  __syncthreads();
  group_sums<PER>(tab, a.vecs, t.lanes, group_width, t.n_groups, [&](int g, float s) { own[g].x = s / count; });
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.0f;
  float m[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) m[j] = own[grp[j]].x;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (!(t.active && t.px0 + t.p + k * t.lanes < t.px1)) continue;
    float x[V::N];
    V::get(raw[k], x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) {
      const float d = x[j] - m[ALIGNED ? 0 : j];
      acc[ALIGNED ? 0 : j] = fmaf(d, d, acc[ALIGNED ? 0 : j]);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) tab[threadIdx.x * PER + j] = acc[j];
  __syncthreads();
  group_sums<PER>(tab, a.vecs, t.lanes, group_width, t.n_groups, [&](int g, float s) { own[g].y = s; });
  if (a.parts > 1) ptx::cluster_sync();
  else __syncthreads();
  const float total = (float)a.pixels * (float)a.cg;
  for (int g = threadIdx.x; g < t.n_groups; g += kNormThreads) {
    float mean = own[g].x, m2 = own[g].y;
    if (a.parts > 1) {
      float2 other[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r >= a.parts) break;
        const uint32_t at = ptx::map_cluster(ptx::smem_u32(&own[g]), (uint32_t)r);
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(other[r].x), "=f"(other[r].y) : "r"(at) : "memory");
      }
      mean = m2 = 0.0f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r >= a.parts) break;
        mean += other[r].x * ((float)(min((r + 1) * a.part_pixels, a.pixels) - r * a.part_pixels) / (float)a.pixels);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r >= a.parts) break;
        const float d = other[r].x - mean, n = (float)(min((r + 1) * a.part_pixels, a.pixels) - r * a.part_pixels) * (float)a.cg;
        m2 += fmaf(d * d, n, other[r].y);
      }
    }
    all[g] = make_float2(mean, rsqrtf(m2 / total + a.eps));
  }
  __syncthreads();
  if (a.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); // the others' numbers have been read
  float r[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    m[j] = all[grp[j]].x;
    r[j] = all[grp[j]].y;
  }
  T *out = (T *)a.out;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int px = t.px0 + t.p + k * t.lanes;
    if (!(t.active && px < t.px1)) continue;
    float x[V::N];
    V::get(raw[k], x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) x[j] = fmaf((x[j] - m[ALIGNED ? 0 : j]) * r[ALIGNED ? 0 : j], ga[j], be[j]);
    activate_all<V::kF32>(a.act, x);
    if (!ALIGNED) {
#pragma unroll
      for (int j = 0; j < V::N; ++j) x[j] = t.ch + j < a.c ? x[j] : 0.0f;
    }
    *reinterpret_cast<uint4 *>(out + t.offset(a, px)) = V::put(x);
  }
  if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // none leaves while its numbers may be read
}

// ---- streamed
template <typename T, bool ALIGNED> __global__ void __launch_bounds__(kNormThreads) group_norm_stats_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  constexpr int PER = ALIGNED ? 1 : V::N;
  extern __shared__ float smem[];
  float *tab = smem;                                                   // [threads][PER]
  float *mean_of = smem + kNormThreads * PER;                          // [groups of the chunk]
  __shared__ int last;
  const NormTile<T> t(a, blockIdx.x);
  pdl_prologue();
  const T *in = (const T *)a.in;
  const int mine = t.active && t.px0 + t.p < t.px1 ? (t.px1 - t.px0 - t.p + t.lanes - 1) / t.lanes : 0;
  // Distances from the first value of each channel (or, where vectors lie within groups, of the vector)
  float first[PER], s[PER], q[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) first[j] = s[j] = q[j] = 0.0f;
  const T *at = in + t.offset(a, t.px0 + t.p);
  const size_t step = (size_t)t.lanes * a.cp;
  auto take = [&](const uint4 &raw) {
    float x[V::N];
    V::get(raw, x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) {
      const int i = ALIGNED ? 0 : j;
      const float d = x[j] - first[i];
      s[i] += d;
      q[i] = fmaf(d, d, q[i]);
    }
  };
  if (mine > 0) {
    float x[V::N];
    V::get(*reinterpret_cast<const uint4 *>(at), x);
#pragma unroll
    for (int j = 0; j < PER; ++j) first[j] = x[j];
  }
  int k = 0;
  for (; k + 8 <= mine; k += 8) {
    uint4 raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const uint4 *>(at + i * step);
    at += 8 * step;
#pragma unroll
    for (int i = 0; i < 8; ++i) take(raw[i]);
  }
  for (; k < mine; ++k, at += step) take(*reinterpret_cast<const uint4 *>(at));
  // per thread: count n, mean = first + s / n, M2 = q - s^2 / n
  const float n = (float)mine * (ALIGNED ? V::N : 1);
  const int group_width = ALIGNED ? a.cg / V::N : a.cg;
  const float count = (float)(t.px1 - t.px0) * (float)a.cg;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (mine > 0) {
      q[j] -= s[j] * (s[j] / n);
      q[j] = q[j] < 0.0f ? 0.0f : q[j]; // (a NaN stays)
      first[j] += s[j] / n;
    }
    tab[threadIdx.x * PER + j] = n * first[j];
  }
  __syncthreads();
  group_sums<PER>(tab, a.vecs, t.lanes, group_width, t.n_groups, [&](int g, float v) { mean_of[g] = v / count; });
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float d = first[j] - mean_of[min((t.ch + j) / a.cg - t.first_group, t.n_groups - 1)];
    tab[threadIdx.x * PER + j] = mine > 0 ? fmaf(n * d, d, q[j]) : 0.0f;
  }
  __syncthreads();
  float2 *partial = a.partial + ((size_t)t.img * a.groups + t.first_group) * a.parts;
  group_sums<PER>(tab, a.vecs, t.lanes, group_width, t.n_groups,
                  [&](int g, float v) { partial[(size_t)g * a.parts + t.part] = make_float2(mean_of[g], v); });
  // the block that comes last joins the parts, in their order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.arrived + t.img * a.chunks + t.chunk, 1u) == (unsigned)a.parts - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int g = threadIdx.x >> 5; g < t.n_groups; g += kNormThreads / 32) {
    const volatile float2 *pp = partial + (size_t)g * a.parts;
    auto share = [&](int r) { return (float)(min((r + 1) * a.part_pixels, a.pixels) - r * a.part_pixels); };
    float mean = 0.0f, m2 = 0.0f;
    for (int r = threadIdx.x & 31; r < a.parts; r += 32) mean += pp[r].x * (share(r) / (float)a.pixels);
    mean = warp_sum(mean);
    for (int r = threadIdx.x & 31; r < a.parts; r += 32) {
      const float d = pp[r].x - mean;
      m2 += fmaf(d * d, share(r) * (float)a.cg, pp[r].y);
    }
    m2 = warp_sum(m2);
    if ((threadIdx.x & 31) == 0)
      a.stats[(size_t)t.img * a.groups + t.first_group + g] = make_float2(mean, rsqrtf(m2 / ((float)a.pixels * (float)a.cg) + a.eps));
  }
  if (threadIdx.x == 0) a.arrived[t.img * a.chunks + t.chunk] = 0u;
}

template <typename T> __global__ void __launch_bounds__(kNormThreads) group_norm_apply_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  const NormTile<T> t(a, gridDim.x - 1 - blockIdx.x);
  float sc[V::N], be[V::N], m[V::N];
  if (t.active) {
    load_floats(a.gamma + t.ch, sc);
    load_floats(a.beta + t.ch, be);
  }
  pdl_prologue();
  if (!t.active) return;
#pragma unroll
  for (int j = 0; j < V::N; ++j) {
    const float2 st = a.stats[(size_t)t.img * a.groups + min((t.ch + j) / a.cg, a.groups - 1)];
    m[j] = st.x;
    sc[j] *= st.y;
  }
  const int mine = t.px0 + t.p < t.px1 ? (t.px1 - t.px0 - t.p + t.lanes - 1) / t.lanes : 0;
  const size_t step = (size_t)t.lanes * a.cp;
  // from the last pixel to the first
  size_t at = t.offset(a, t.px0 + t.p) + (size_t)max(mine - 1, 0) * step;
  const T *in = (const T *)a.in;
  T *out = (T *)a.out;
  auto put = [&](const uint4 &raw, size_t o) {
    float x[V::N];
    V::get(raw, x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) x[j] = fmaf(x[j] - m[j], sc[j], be[j]);
    activate_all<V::kF32>(a.act, x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) x[j] = t.ch + j < a.c ? x[j] : 0.0f;
    *reinterpret_cast<uint4 *>(out + o) = V::put(x);
  };
  int k = 0;
  for (; k + 4 <= mine; k += 4) {
    uint4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = *reinterpret_cast<const uint4 *>(in + at - i * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) put(raw[i], at - i * step);
    at -= 4 * step;
  }
  for (; k < mine; ++k, at -= step) put(*reinterpret_cast<const uint4 *>(in + at), at);
}

// ---- strided: one block per image and group, three passes over its values
template <typename T> __global__ void group_norm_strided_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
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
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) s += V::one(in[at(i)]);
  const float mean = block_sum(s, red) / (float)count;
  s = 0.0f;
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) {
    const float d = V::one(in[at(i)]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = rsqrtf(block_sum(s, red) / (float)count + a.eps);
  for (size_t i = threadIdx.x; i < count; i += blockDim.x) {
    const size_t o = at(i);
    const int ch = g * a.cg + (int)(o % a.cp);
    float v[1] = {fmaf((V::one(in[o]) - mean) * rstd, a.gamma[ch], a.beta[ch])};
    activate_all<V::kF32>(a.act, v);
    out[o] = V::back(v[0]);
  }
}

inline void launch_group_norm(const GroupNormArgs &a, const GroupNormPlan &p, bool f32, cudaStream_t s) {
  auto by_type = [&](auto type) {
    typedef decltype(type) T;
    auto by_nv = [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if (p.form == NORM_ROWS_WARP) launch_k(group_norm_rows_kernel<T, NV, false>, p.grid, 128, 0, s, a);
      else if constexpr (NV <= 4) launch_k(group_norm_rows_kernel<T, NV, true>, p.grid, p.threads, 0, s, a);
    };
    auto slab_nv = [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if (p.aligned) launch_cluster_k(a.parts, group_norm_slab_kernel<T, true, NV>, p.grid, kNormThreads, p.smem, s, a);
      else launch_cluster_k(a.parts, group_norm_slab_kernel<T, false, NV>, p.grid, kNormThreads, p.smem, s, a);
    };
    switch (p.form) {
    case NORM_ROWS_WARP:
    case NORM_ROWS_BLOCK:
      if (p.nv <= 1) by_nv(std::integral_constant<int, 1>());
      else if (p.nv <= 2) by_nv(std::integral_constant<int, 2>());
      else if (p.nv <= 4) by_nv(std::integral_constant<int, 4>());
      else by_nv(std::integral_constant<int, 8>());
      break;
    case NORM_SLAB:
      if (p.nv <= 2) slab_nv(std::integral_constant<int, 2>());
      else if (p.nv <= 4) slab_nv(std::integral_constant<int, 4>());
      else if (p.nv <= 8) slab_nv(std::integral_constant<int, 8>());
      else slab_nv(std::integral_constant<int, 16>());
      break;
    case NORM_STREAMED:
      if (p.aligned) launch_k(group_norm_stats_kernel<T, true>, p.grid, kNormThreads, p.smem, s, a);
      else launch_k(group_norm_stats_kernel<T, false>, p.grid, kNormThreads, p.smem, s, a);
      launch_k(group_norm_apply_kernel<T>, p.grid, kNormThreads, 0, s, a);
      break;
    default: launch_k(group_norm_strided_kernel<T>, p.grid, kNormThreads, 0, s, a);
    }
  };
  if (f32) by_type(float());
  else by_type(uint16_t());
}

} // namespace tpucb
