// Group normalisation with an activation, channels last: per image n and group g of c / groups neighbouring channels
//   mean = E[x], var = E[(x - mean)^2] over the image's pixels and the group's channels,
//   y = act((x - mean) / sqrt(var + eps) * gamma[channel] + beta[channel]).
// groups = 1 on a [tokens, channels] tensor is layer norm. Statistics and affine in fp32, one rounding at the end. Bound: memory,
// x read and y written once.
//
// Four forms (group_norm_plan), threads moving vectors of 16 bytes:
//   rows     one pixel per image: a group is contiguous; a warp or a block keeps it in registers;
//   slab     the pixels of an image x a few groups ("chunk") are kept in the shared memory of a cluster of up to eight blocks, which
//            exchange their statistics through it: x is read once;
//   streamed larger ones: a pass for the statistics of parts of an image, and a pass that joins them and forms the results, in the
//            opposite order, so that it begins with what the L2 still holds;
//   strided  the same two passes, value by value: images where the smallest run of whole groups that is also whole vectors has more than 256
//            vectors and does not fit a slab, or more than 512 (2 x 2560 x 32 x 32 in one group: 320 vectors).
// Rows take the mean first and then the squares of the distances from it, out of the registers. The other forms sum, in one pass, the distances
// from the first value that a thread sees (in a channel, or in all of its vectors where they lie within a group) and their squares, and take
// q - s s / n: a difference, whose error is at most 2 (L + 4) (L + 1) 2^-24 of the variance for the L values that a thread sums one after the other, also
// where the first value is an outlier, which is part of the variance itself. (One such value for the whole block cost 1e-4 of it.) Partial ones are joined
// without differences of sums:
//   M2 = sum M2_i + sum n_i (mean_i - mean)^2.
// The result is one multiply-add per value, with beta - mean rstd gamma rounded once. Its error is like that of the mean itself, a few 2^-24 |mean| rstd
// gamma: in a group of equal values c, whose rstd is 1 / sqrt(eps), beta is met to that (c = 10, eps = 1e-5: 6e-5), as in a plain fp32
// form whose mean is rounded.
#pragma once
#include "activation.cuh"
#include "conv_plan.cuh"

namespace tpucb {

struct GroupNormArgs {
  const void *in;
  void *out;
  const float *gamma, *beta; // [cp], zero behind c
  int n, pixels, c, cp, groups, cg;
  float eps;
  int act;
  // slab and streamed: chunks of `vecs` vectors = whole groups (the last may have fewer), `parts` blocks share an image's pixels
  int held; // slab: vectors per thread
  int vecs, lanes, chunk_groups, chunks, parts, part_pixels; // (lanes: pixels that a block's threads take at once)
  int apply_parts, apply_pixels; // streamed: of the second pass
  long long part_values;         // strided: of a group, per block
  int col_split, group_span;     // norm_group_sums: threads per column; parts of columns per group, rounded up to whole warps
  float inv_vecs, inv_lanes, inv_cg, inv_width, inv_group_width;        // 1 / vecs and so on, for quotients of small numbers (small_div)
  float2 *partial;               // streamed: [n][groups][parts] mean, M2
};
// a / b for a < 2^22, given 1 / b: a + 1/2 is at least 1 / (2 b) of a quotient away from the next whole one, and the product's error less
__device__ __forceinline__ int small_div(int a, float inv_b) { return (int)(((float)a + 0.5f) * inv_b); }

// Sixteen bytes of values, as pairs
template <typename T> struct NormVec;
template <> struct NormVec<float> {
  static constexpr int N = 4, P = 2;
  static constexpr bool kF32 = true;
  static __device__ __forceinline__ void get(const uint4 &r, Pair (&v)[2]) {
    v[0] = Pair(__uint_as_float(r.x), __uint_as_float(r.y));
    v[1] = Pair(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  static __device__ __forceinline__ uint4 put(const Pair (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].lo()), __float_as_uint(v[0].hi()), __float_as_uint(v[1].lo()), __float_as_uint(v[1].hi()));
  }
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float back(float v) { return v; }
};
template <> struct NormVec<uint16_t> {
  static constexpr int N = 8, P = 4;
  static constexpr bool kF32 = false;
  static __device__ __forceinline__ void get(const uint4 &r, Pair (&v)[4]) {
    v[0] = pair_of_bf16(r.x);
    v[1] = pair_of_bf16(r.y);
    v[2] = pair_of_bf16(r.z);
    v[3] = pair_of_bf16(r.w);
  }
  static __device__ __forceinline__ uint4 put(const Pair (&v)[4]) {
    return make_uint4(bf16x2_ieee(v[0].lo(), v[0].hi()), bf16x2_ieee(v[1].lo(), v[1].hi()), bf16x2_ieee(v[2].lo(), v[2].hi()),
                      bf16x2_ieee(v[3].lo(), v[3].hi()));
  }
  static __device__ __forceinline__ float one(uint16_t v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ uint16_t back(float v) { return (uint16_t)bf16x2_ieee(v, v); }
};

template <int ACT, bool F32, int P> __device__ __forceinline__ void activate_all(Pair (&v)[P]) {
#pragma unroll
  for (int j = 0; j < P; ++j) v[j] = activate<ACT, F32>(v[j]);
}
template <int P> __device__ __forceinline__ void load_floats(const float *p, Pair (&v)[P]) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    const float4 f = __ldg(reinterpret_cast<const float4 *>(p) + i);
    v[2 * i] = Pair(f.x, f.y);
    v[2 * i + 1] = Pair(f.z, f.w);
  }
}
// 16 bytes that this SM reads once: they take no place in its L1 (statistics pass of 1 x 256 x 512 x 512 30.5 -> 23.6 us)
__device__ __forceinline__ uint4 load_once(const void *p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}
// zero behind the first `valid` values
template <int P> __device__ __forceinline__ void clip(Pair (&v)[P], int valid) {
#pragma unroll
  for (int j = 0; j < P; ++j) v[j] = Pair(2 * j < valid ? v[j].lo() : 0.0f, 2 * j + 1 < valid ? v[j].hi() : 0.0f);
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

// ---- rows: groups of one pixel. LANES: 8 or 32 lanes of a warp per R groups, 0: a block. NV: vectors per thread. FULL: every thread has that
// many, of channels only; the threads' means and squares are then joined in one exchange instead of two.
// gamma and beta are four times the bytes of a BF16 vector: with one row at a time the L1's data path was 61% busy (4099 x 4096: 15.0 us with
// three modules in flight, with two 13.9, 4.8 TB/s: bound by memory, with one set of loads per block to hide it).
template <typename T, int NV, int R, int LANES, bool FULL> __global__ void __launch_bounds__(LANES ? 128 : 512) group_norm_rows_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  constexpr bool BLOCK = LANES == 0;
  __shared__ float2 red[R][16];
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & (LANES - 1), lanes = BLOCK ? blockDim.x : LANES;
  const int unit = BLOCK ? blockIdx.x : blockIdx.x * (128 / (BLOCK ? 1 : LANES)) + threadIdx.x / (BLOCK ? 1 : LANES); // R images, one of their groups
  pdl_prologue();
  const int nvec = (a.cg + V::N - 1) / V::N;
  // (without FULL the first half of the vectors is there all the same: plan)
  auto has = [&](int k) { return FULL || k < NV / 2 || lane + k * lanes < nvec; };
  const bool tail = !FULL && a.cg % V::N; // the last vector ends in padded channels, which count as zero
  auto cut = [&](Pair (&x)[V::P], int k) {
    if (k >= NV / 2 && tail && lane + k * lanes == nvec - 1) clip(x, a.cg - (lane + k * lanes) * V::N);
  };
  const int images = a.groups == 1 ? unit : unit / a.groups, g = unit - images * a.groups, img0 = images * R;
  auto offset = [&](int r) { return (size_t)(img0 + r) * a.cp + (size_t)g * a.cg + (size_t)lane * V::N; };
  uint4 raw[R][NV];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint4 *in = reinterpret_cast<const uint4 *>((const T *)a.in + offset(r));
#pragma unroll
    for (int k = 0; k < NV; ++k) raw[r][k] = has(k) && img0 + r < a.n ? load_once(in + k * lanes) : make_uint4(0u, 0u, 0u, 0u);
  }
  float mean[R], m2[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    Pair s = both(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      Pair x[V::P];
      V::get(raw[r][k], x);
      cut(x, k);
#pragma unroll
      for (int j = 0; j < V::P; ++j) s = s + x[j];
    }
    mean[r] = (s.lo() + s.hi()) * (FULL ? 1.0f / (NV * V::N) : a.inv_cg);
  }
  const int warps = blockDim.x >> 5;
  // sums over the block (or the warp) of one number per row
  auto join = [&](float (&v)[R]) {
#pragma unroll
    for (int o = 1; o < (BLOCK ? 32 : LANES); o *= 2)
#pragma unroll
      for (int r = 0; r < R; ++r) v[r] += __shfl_xor_sync(0xffffffffu, v[r], o);
    if (BLOCK) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) red[r][threadIdx.x >> 5].x = v[r];
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        v[r] = 0.0f;
        for (int w = 0; w < warps; ++w) v[r] += red[r][w].x;
      }
    }
  };
  if (!FULL) join(mean);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    Pair s = both(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!has(k)) continue;
      Pair x[V::P];
      V::get(raw[r][k], x);
#pragma unroll
      for (int j = 0; j < V::P; ++j) x[j] = x[j] + both(-mean[r]);
      cut(x, k);
#pragma unroll
      for (int j = 0; j < V::P; ++j) s = fma(x[j], x[j], s);
    }
    m2[r] = s.lo() + s.hi();
  }
  if (FULL) {
    // equal counts: the mean of two is half their sum, and their M2 grows by half the count times the square of the distance
    float half = 0.5f * NV * V::N;
#pragma unroll
    for (int o = 1; o < (BLOCK ? 32 : LANES); o *= 2) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float other = __shfl_xor_sync(0xffffffffu, mean[r], o), d = mean[r] - other;
        m2[r] += __shfl_xor_sync(0xffffffffu, m2[r], o);
        m2[r] = fmaf(d * half, d, m2[r]);
        mean[r] = 0.5f * (mean[r] + other);
      }
      half *= 2.0f;
    }
    if (BLOCK) {
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) red[r][threadIdx.x >> 5] = make_float2(mean[r], m2[r]);
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        mean[r] = m2[r] = 0.0f;
        for (int w = 0; w < warps; ++w) mean[r] += red[r][w].x;
        mean[r] *= 1.0f / (float)warps;
        for (int w = 0; w < warps; ++w) {
          const float2 o = red[r][w];
          m2[r] += fmaf((o.x - mean[r]) * (32.0f * NV * V::N), o.x - mean[r], o.y);
        }
      }
    }
  } else {
    join(m2);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m2[r] = rsqrtf(fmaf(m2[r], a.inv_cg, a.eps));
    mean[r] *= -m2[r];
  }
  const float *gamma = a.gamma + g * a.cg + lane * V::N, *beta = a.beta + g * a.cg + lane * V::N;
  with_activation(a.act, [&](auto act) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!has(k)) continue;
      Pair ga[V::P], be[V::P];
      load_floats(gamma + k * lanes * V::N, ga);
      load_floats(beta + k * lanes * V::N, be);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Pair x[V::P];
        V::get(raw[r][k], x);
#pragma unroll
        for (int j = 0; j < V::P; ++j) x[j] = fma(fma(x[j], both(m2[r]), both(mean[r])), ga[j], be[j]);
        activate_all<decltype(act)::value, V::kF32>(x);
        cut(x, k);
        if (img0 + r < a.n) reinterpret_cast<uint4 *>((T *)a.out + offset(r))[k * lanes] = V::put(x);
      }
    }
  });
}

// ---- what slab and streamed share: a block takes pixels x a chunk; a thread keeps to one vector column
template <typename T, int THREADS> struct NormTile { // (parts: of the image, of `pixels` each)
  int img, chunk, part, first_group, n_groups; // groups of this chunk
  int px0, px1;                                // this block's pixels
  int v, p, lanes, ch;                         // the thread's vector column, pixel lane, pixel lanes of the block, first channel
  bool active;
  __device__ __forceinline__ NormTile(const GroupNormArgs &a, unsigned block, int parts, int pixels) {
    const int slab = parts == 1 ? block : block / parts;
    part = block - slab * parts;
    img = a.chunks == 1 ? slab : slab / a.chunks;
    chunk = slab - img * a.chunks; // (chunks of a pixel that share a line of the L2 are neighbours in the grid)
    first_group = chunk * a.chunk_groups;
    n_groups = min(a.chunk_groups, a.groups - first_group);
    px0 = part * pixels;
    px1 = min(px0 + pixels, a.pixels);
    lanes = a.lanes;
    p = small_div(threadIdx.x, a.inv_vecs);
    v = threadIdx.x - p * a.vecs;
    ch = (chunk * a.vecs + v) * NormVec<T>::N;
    active = p < lanes && ch < a.c;
  }
  __device__ __forceinline__ size_t offset(const GroupNormArgs &a, int px) const { return ((size_t)img * a.pixels + px) * a.cp + ch; }
};
// The block's sum over each group of its chunk of what the threads hold per channel or, where vectors lie within groups (ALIGNED), in
// all: `done(group of the chunk, sum)` in one thread each. Three short steps, as these sums are what small tensors take their time for
// (with a warp per group and a loop over all of its values, 2 x 1280 x 8 x 8 took 3.4 us instead of 2.2): columns (vectors or channels)
// over the pixel lanes, several threads per column; warps over 32 of a group's column parts; groups over their warps' sums.
// tab: THREADS x PER floats, then a.group_span per group, then that / 32; the parts behind a group's last are zero (norm_clear).
template <typename T, bool ALIGNED, int THREADS, class Done>
__device__ __forceinline__ void norm_group_sums(const GroupNormArgs &a, const NormTile<T, THREADS> &t, const Pair *x, float *tab, Done done) {
  typedef NormVec<T> V;
  constexpr int PER = ALIGNED ? 1 : V::N;
  const int width = a.vecs * PER, group_width = ALIGNED ? a.cg / V::N : a.cg;
  float *cols = tab + THREADS * PER, *warps = cols + a.chunk_groups * a.group_span;
  if constexpr (ALIGNED) {
    tab[threadIdx.x] = x[0].lo() + x[0].hi();
  } else {
#pragma unroll
    for (int j = 0; j < V::P; ++j) *reinterpret_cast<float2 *>(tab + threadIdx.x * PER + 2 * j) = make_float2(x[j].lo(), x[j].hi());
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.col_split * width; i += THREADS) {
    const int part = a.col_split == 1 ? 0 : small_div(i, a.inv_width), col = i - part * width, g = small_div(col, a.inv_group_width);
    float s = 0.0f;
#pragma unroll 4
    for (int p = part; p < t.lanes; p += a.col_split) s += tab[p * width + col];
    if (g < t.n_groups) cols[g * a.group_span + part * group_width + col - g * group_width] = s;
  }
  __syncthreads();
  const int span = a.group_span >> 5; // warps' sums per group
  for (int b = threadIdx.x >> 5; b < t.n_groups * span; b += THREADS / 32) {
    const float s = warp_sum(cols[b * 32 + (threadIdx.x & 31)]);
    if ((threadIdx.x & 31) == 0) warps[b] = s;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < t.n_groups; g += THREADS) {
    float s = 0.0f;
#pragma unroll 4
    for (int b = 0; b < span; ++b) s += warps[g * span + b];
    done(g, s);
  }
}
// before the first norm_group_sums (whose barriers order it)
template <typename T, bool ALIGNED, int THREADS> __device__ __forceinline__ void norm_clear(const GroupNormArgs &a, float *tab) {
  float *cols = tab + THREADS * (ALIGNED ? 1 : NormVec<T>::N);
  for (int i = threadIdx.x; i < a.chunk_groups * a.group_span; i += THREADS) cols[i] = 0.0f;
}
// Calls use(j, group of channel ch + j, of the image) for the channels of a vector, behind the last group the last one.
template <int N, class Use> __device__ __forceinline__ void for_groups(const GroupNormArgs &a, int ch, Use use) {
  int g = small_div(ch, a.inv_cg), left = (g + 1) * a.cg - ch;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    use(j, min(g, a.groups - 1));
    if (--left == 0) {
      ++g;
      left = a.cg;
    }
  }
}
// minus the mean of each channel's group; mean(group of the chunk)
template <typename T, bool ALIGNED, class Mean>
__device__ __forceinline__ void own_means(const GroupNormArgs &a, int ch, int first_group, int n_groups, Mean mean, Pair *m) {
  if (ALIGNED) {
    m[0] = both(-mean(min(small_div(ch, a.inv_cg) - first_group, n_groups - 1)));
  } else {
    float v[NormVec<T>::N];
    for_groups<NormVec<T>::N>(a, ch, [&](int j, int g) { v[j] = -mean(min(g - first_group, n_groups - 1)); });
#pragma unroll
    for (int j = 0; j < NormVec<T>::P; ++j) m[j] = Pair(v[2 * j], v[2 * j + 1]);
  }
}
// What a thread of a slab sums: distances from its first value and their squares, per channel or, where vectors lie within groups, in all.
template <typename T, bool ALIGNED> constexpr int kMoments = ALIGNED ? 1 : NormVec<T>::P;
template <typename T, bool ALIGNED> __device__ __forceinline__ void moments_take(const uint4 &raw, const Pair *first, Pair *s, Pair *q) { // first: negative
  Pair x[NormVec<T>::P];
  NormVec<T>::get(raw, x);
#pragma unroll
  for (int j = 0; j < NormVec<T>::P; ++j) {
    const int i = ALIGNED ? 0 : j;
    const Pair d = x[j] + first[i];
    s[i] = s[i] + d;
    q[i] = fma(d, d, q[i]);
  }
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void moments_begin(const uint4 &raw, Pair *first) {
  Pair x[NormVec<T>::P];
  NormVec<T>::get(raw, x);
#pragma unroll
  for (int j = 0; j < kMoments<T, ALIGNED>; ++j) first[j] = ALIGNED ? both(-x[0].lo()) : x[j] * both(-1.0f);
}
// The block's mean and M2 of each group of its chunk, from `mine` vectors of each thread: `done(group of the chunk, mean, M2)` in one thread
// each. mean_of: [groups of the chunk]; tab: norm_group_sums. (Where vectors lie within groups both halves of the pairs count as columns.)
template <typename T, bool ALIGNED, int THREADS, class Done>
__device__ __forceinline__ void moments_join(const GroupNormArgs &a, const NormTile<T, THREADS> &t, int mine, Pair *first, const Pair *s, Pair *q, float *mean_of,
                                             float *tab, Done done) {
  constexpr int P = kMoments<T, ALIGNED>;
  const float n = (float)mine * (ALIGNED ? NormVec<T>::P : 1), inv = mine > 0 ? 1.0f / n : 0.0f;
  const float inv_count = 1.0f / ((float)(t.px1 - t.px0) * (float)a.cg);
  Pair x[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const Pair mean = s[j] * both(inv);
    q[j] = fma(s[j] * both(-1.0f), mean, q[j]);
    q[j] = Pair(q[j].lo() < 0.0f ? 0.0f : q[j].lo(), q[j].hi() < 0.0f ? 0.0f : q[j].hi()); // (a NaN stays)
    first[j] = fma(first[j], both(-1.0f), mean); // the mean
    x[j] = first[j] * both(n);
  }
  norm_group_sums<T, ALIGNED, THREADS>(a, t, x, tab, [&](int g, float sum) { mean_of[g] = sum * inv_count; });
  __syncthreads();
  Pair m[P];
  own_means<T, ALIGNED>(a, t.ch, t.first_group, t.n_groups, [&](int g) { return mean_of[g]; }, m);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const Pair d = first[j] + m[j];
    x[j] = mine > 0 ? fma(d * both(n), d, q[j]) : both(0.0f);
  }
  norm_group_sums<T, ALIGNED, THREADS>(a, t, x, tab, [&](int g, float sum) { done(g, mean_of[g], sum); });
}
// y = x scale + shift of a thread's channels
template <typename T> struct NormAffine {
  typedef NormVec<T> V;
  Pair scale[V::P], shift[V::P];
  __device__ __forceinline__ void load(const GroupNormArgs &a, int ch) {
    load_floats(a.gamma + ch, scale);
    load_floats(a.beta + ch, shift);
  }
  // `stat(group of the image)`: mean and 1 / sqrt(var + eps)
  template <bool ALIGNED, class Stat> __device__ __forceinline__ void set(const GroupNormArgs &a, int ch, Stat stat) {
    if (ALIGNED) {
      const float2 st = stat(small_div(ch, a.inv_cg));
#pragma unroll
      for (int j = 0; j < V::P; ++j) {
        scale[j] = scale[j] * both(st.y);
        shift[j] = fma(both(-st.x), scale[j], shift[j]);
      }
    } else {
      float2 st[V::N];
      for_groups<V::N>(a, ch, [&](int j, int g) { st[j] = stat(g); });
#pragma unroll
      for (int j = 0; j < V::P; ++j) {
        scale[j] = scale[j] * Pair(st[2 * j].y, st[2 * j + 1].y);
        shift[j] = fma(Pair(-st[2 * j].x, -st[2 * j + 1].x), scale[j], shift[j]);
      }
    }
  }
  template <int ACT> __device__ __forceinline__ uint4 apply(const uint4 &raw, int valid) const {
    Pair x[V::P];
    V::get(raw, x);
#pragma unroll
    for (int j = 0; j < V::P; ++j) x[j] = fma(x[j], scale[j], shift[j]);
    activate_all<ACT, V::kF32>(x);
    if (valid < V::N) clip(x, valid);
    return V::put(x);
  }
};

// ---- slab. ALIGNED: a vector's channels belong to one group. A thread's vectors wait in shared memory, [vector][thread], where it alone writes
// and reads them: no barrier orders them. Bound by the memory's latency and the sums between its two halves, which other blocks of the SM fill where
// there are any: 64 x 256 x 32 x 32 with SiLU 14.8 us with three modules in flight (69% of the memory's rate), 8 x 320 x 64 x 64 12.8, one
// module's launches behind one another 18.5. (With the vectors in registers, eight per thread, those took 22.8, 25.1 and 28.7 us: a wave of blocks held half as much, in one block
// per SM.)
template <typename T, bool ALIGNED, int THREADS> __global__ void __launch_bounds__(THREADS, 1024 / THREADS) group_norm_slab_kernel(const GroupNormArgs a) {
  extern __shared__ __align__(16) float smem[];
  uint4 *held = reinterpret_cast<uint4 *>(smem) + threadIdx.x;
  float2 *own = reinterpret_cast<float2 *>(smem + (size_t)a.held * THREADS * 4); // [groups of the chunk]: this block's mean and M2
  float2 *all = own + a.chunk_groups;                                                 // mean and 1 / sqrt(var + eps) of the image
  float *tab = reinterpret_cast<float *>(all + a.chunk_groups);
  const NormTile<T, THREADS> t(a, blockIdx.x, a.parts, a.part_pixels);
  const size_t at = t.offset(a, t.px0 + t.p), step = (size_t)t.lanes * a.cp;
  const int mine = t.active && t.px0 + t.p < t.px1 ? small_div(t.px1 - t.px0 - t.p + t.lanes - 1, a.inv_lanes) : 0;
  norm_clear<T, ALIGNED, THREADS>(a, tab);
  pdl_prologue();
  {
    const T *in = (const T *)a.in + at;
    uint32_t to = ptx::smem_u32(held);
#pragma unroll 4
    for (int k = 0; k < mine; ++k, in += step, to += THREADS * 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(in) : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  constexpr int P = kMoments<T, ALIGNED>;
  Pair first[P], sum[P], square[P];
#pragma unroll
  for (int j = 0; j < P; ++j) first[j] = sum[j] = square[j] = both(0.0f);
  if (mine > 0) {
    moments_begin<T, ALIGNED>(held[0], first);
#pragma unroll 4
    for (int k = 0; k < mine; ++k) moments_take<T, ALIGNED>(held[k * THREADS], first, sum, square);
  }
  float *mean_of = reinterpret_cast<float *>(all);
  moments_join<T, ALIGNED>(a, t, mine, first, sum, square, mean_of, tab, [&](int g, float mean, float m2) { own[g] = make_float2(mean, m2); });
  NormAffine<T> affine;
  if (t.active) affine.load(a, t.ch);
  if (a.parts > 1) ptx::cluster_sync();
  else __syncthreads();
  const float total = (float)a.pixels * (float)a.cg;
  if (a.parts == 1) {
    for (int g = threadIdx.x; g < t.n_groups; g += THREADS) all[g] = make_float2(own[g].x, rsqrtf(own[g].y / total + a.eps));
  } else {
    // eight threads per group, one block's numbers each (a thread that read them all took a round trip for each: 2 x 320 x 96 x 96 by 8
    // blocks 12.7 us with three modules in flight instead of 11.3)
    const int r = threadIdx.x & 7;
    const float share = r < a.parts ? (float)(min((r + 1) * a.part_pixels, a.pixels) - r * a.part_pixels) : 0.0f;
    auto sum8 = [](float v) {
#pragma unroll
      for (int k = 4; k; k /= 2) v += __shfl_xor_sync(0xffffffffu, v, k);
      return v;
    };
    for (int first = 0; first < t.n_groups; first += THREADS / 8) {
      const int g = min(first + (int)threadIdx.x / 8, t.n_groups - 1);
      float2 o = make_float2(0.0f, 0.0f);
      if (r < a.parts)
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(o.x), "=f"(o.y) : "r"(ptx::map_cluster(ptx::smem_u32(&own[g]), (uint32_t)r)) : "memory");
      const float mean = sum8(o.x * (share / (float)a.pixels)), d = o.x - mean;
      const float m2 = sum8(r < a.parts ? fmaf(d * d, share * (float)a.cg, o.y) : 0.0f);
      if (r == 0) all[g] = make_float2(mean, rsqrtf(m2 / total + a.eps)); // (several threads of the last group write the same)
    }
  }
  __syncthreads();
  if (a.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); // the others' numbers have been read
  if (t.active) {
    affine.template set<ALIGNED>(a, t.ch, [&](int g) { return all[g - t.first_group]; });
    T *out = (T *)a.out;
    const int valid = ALIGNED ? NormVec<T>::N : a.c - t.ch;
    with_activation(a.act, [&](auto act) {
#pragma unroll 2
      for (int k = 0; k < mine; ++k)
        *reinterpret_cast<uint4 *>(out + at + k * step) = affine.template apply<decltype(act)::value>(held[k * THREADS], valid);
    });
  }
  __syncwarp();
  if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // none leaves while its numbers may be read
}

// ---- streamed
// use(vector, index) for `count` vectors that are `step` values apart, the next D of them on their way while D are used (with one set of
// four and no way ahead: 4 x 128 x 128 x 128 12.3 us with three modules in flight instead of 10.7, fp32 2 x 100 x 400 x 400 165 instead of 70).
template <int D, typename T, class Use> __device__ __forceinline__ void for_vectors(const T *p, long long step, int count, Use use) {
  uint4 r[2][D];
  auto fetch = [&](uint4 (&to)[D], int k) {
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (k + i < count) to[i] = load_once(p + (k + i) * step);
  };
  auto each = [&](const uint4 (&from)[D], int k) {
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (k + i < count) use(from[i], k + i);
  };
  fetch(r[0], 0);
  for (int k = 0; k < count; k += 2 * D) {
    fetch(r[1], k + D);
    each(r[0], k);
    fetch(r[0], k + 2 * D);
    each(r[1], k + D);
  }
}

// The slab's sums, written out: through moments_join the compiled loop is slower where groups are no whole vectors (6 x 320 x 128 x 128 46.4 us with
// three modules in flight instead of 38.9; the registers are the same).
template <typename T, bool ALIGNED> __global__ void __launch_bounds__(kStreamThreads, 3) group_norm_stats_kernel(const GroupNormArgs a) {
  extern __shared__ float smem[];
  const NormTile<T, kStreamThreads> t(a, blockIdx.x, a.parts, a.part_pixels);
  float *mean_of = smem; // [groups of the chunk]
  float *tab = smem + (a.chunk_groups + 1) / 2 * 2;
  norm_clear<T, ALIGNED, kStreamThreads>(a, tab);
  pdl_prologue();
  const int mine = t.active && t.px0 + t.p < t.px1 ? small_div(t.px1 - t.px0 - t.p + t.lanes - 1, a.inv_lanes) : 0;
  typedef NormVec<T> V;
  constexpr int P = ALIGNED ? 1 : V::P;
  Pair first[P], s[P], q[P]; // first: negative
#pragma unroll
  for (int j = 0; j < P; ++j) first[j] = s[j] = q[j] = both(0.0f);
  auto take = [&](const uint4 &raw) {
    Pair x[V::P];
    V::get(raw, x);
#pragma unroll
    for (int j = 0; j < V::P; ++j) {
      const int i = ALIGNED ? 0 : j;
      const Pair d = x[j] + first[i];
      s[i] = s[i] + d;
      q[i] = fma(d, d, q[i]);
    }
  };
  if (mine > 0) {
    const T *at = (const T *)a.in + t.offset(a, t.px0 + t.p);
    const size_t step = (size_t)t.lanes * a.cp;
    {
      Pair x[V::P];
      V::get(*reinterpret_cast<const uint4 *>(at), x);
#pragma unroll
      for (int j = 0; j < P; ++j) first[j] = ALIGNED ? both(-x[0].lo()) : x[j] * both(-1.0f);
    }
    for_vectors<ALIGNED ? 4 : 2>(at, (long long)step, mine, [&](const uint4 &raw, int) { take(raw); });
  }
  // The thread's count, mean and M2 (per channel; where vectors lie within groups both halves count as columns of their own)
  const float n = (float)mine * (ALIGNED ? V::P : 1), inv = mine > 0 ? 1.0f / n : 0.0f;
  const float inv_count = 1.0f / ((float)(t.px1 - t.px0) * (float)a.cg);
  Pair x[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const Pair mean = s[j] * both(inv);
    q[j] = fma(s[j] * both(-1.0f), mean, q[j]);
    q[j] = Pair(q[j].lo() < 0.0f ? 0.0f : q[j].lo(), q[j].hi() < 0.0f ? 0.0f : q[j].hi()); // (a NaN stays)
    first[j] = fma(first[j], both(-1.0f), mean); // the mean
    x[j] = first[j] * both(n);
  }
  norm_group_sums<T, ALIGNED, kStreamThreads>(a, t, x, tab, [&](int g, float sum) { mean_of[g] = sum * inv_count; });
  __syncthreads();
  Pair m[P];
  own_means<T, ALIGNED>(a, t.ch, t.first_group, t.n_groups, [&](int g) { return mean_of[g]; }, m);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const Pair d = first[j] + m[j];
    x[j] = mine > 0 ? fma(d * both(n), d, q[j]) : both(0.0f);
  }
  float2 *partial = a.partial + ((size_t)t.img * a.groups + t.first_group) * a.parts;
  norm_group_sums<T, ALIGNED, kStreamThreads>(a, t, x, tab, [&](int g, float sum) { partial[(size_t)g * a.parts + t.part] = make_float2(mean_of[g], sum); });
}

template <typename T, bool ALIGNED> __global__ void __launch_bounds__(kStreamThreads, 3) group_norm_apply_kernel(const GroupNormArgs a) {
  extern __shared__ float smem[];
  float2 *stats = reinterpret_cast<float2 *>(smem); // [groups of the chunk]: mean, 1 / sqrt(var + eps)
  const NormTile<T, kStreamThreads> t(a, gridDim.x - 1 - blockIdx.x, a.apply_parts, a.apply_pixels);
  NormAffine<T> affine;
  if (t.active) affine.load(a, t.ch);
  pdl_prologue();
  // the parts, in their order: a warp per group
  const float inv_pixels = 1.0f / (float)a.pixels, cg = (float)a.cg;
  auto share = [&](int r) { return (float)(min((r + 1) * a.part_pixels, a.pixels) - r * a.part_pixels); };
  for (int g = threadIdx.x >> 5; g < t.n_groups; g += kStreamThreads / 32) {
    const float2 *partial = a.partial + ((size_t)t.img * a.groups + t.first_group + g) * a.parts;
    const int lane = threadIdx.x & 31;
    float mean = 0.0f, m2 = 0.0f;
#pragma unroll 4
    for (int r = lane; r < a.parts; r += 32) mean += partial[r].x * (share(r) * inv_pixels);
    mean = warp_sum(mean);
#pragma unroll 4
    for (int r = lane; r < a.parts; r += 32) {
      const float2 o = partial[r];
      m2 += fmaf((o.x - mean) * (o.x - mean), share(r) * cg, o.y);
    }
    m2 = warp_sum(m2);
    if (lane == 0) stats[g] = make_float2(mean, rsqrtf(m2 * inv_pixels / cg + a.eps));
  }
  __syncthreads();
  if (!t.active) return;
  affine.template set<ALIGNED>(a, t.ch, [&](int g) { return stats[g - t.first_group]; });
  const int mine = t.px0 + t.p < t.px1 ? small_div(t.px1 - t.px0 - t.p + t.lanes - 1, a.inv_lanes) : 0, valid = ALIGNED ? NormVec<T>::N : a.c - t.ch;
  const size_t step = (size_t)t.lanes * a.cp;
  // from the last pixel to the first
  const size_t at = t.offset(a, t.px0 + t.p) + (size_t)max(mine - 1, 0) * step;
  T *out = (T *)a.out + at;
  with_activation(a.act, [&](auto act) {
    for_vectors<4>((const T *)a.in + at, -(long long)step, mine, [&](const uint4 &raw, int k) {
      *reinterpret_cast<uint4 *>(out - k * step) = affine.template apply<decltype(act)::value>(raw, valid);
    });
  });
}

// ---- strided: groups of any width, value by value, a block per part of a group; statistics and results as in the streamed form. Bound by its
// instructions: 2 x 2560 x 32 x 32 with one group 16.3 us with three modules in flight (20% of the memory's rate), one module's launches behind one
// another 27.6 (one block per group 5525).
template <typename T, class Use> __device__ __forceinline__ void for_group_values(const GroupNormArgs &a, Use use) { // use(offset, channel)
  const unsigned lot = blockIdx.x / a.parts, part = blockIdx.x - lot * a.parts, img = lot / a.groups, g = lot - img * a.groups;
  const long long from = part * a.part_values, to = min(from + a.part_values, (long long)a.pixels * a.cg);
  if (from + threadIdx.x >= to) return;
  long long left = (to - from - threadIdx.x + blockDim.x - 1) / blockDim.x, px = (from + threadIdx.x) / a.cg;
  int ch = (int)(from + threadIdx.x - px * a.cg);
  const int step_px = blockDim.x / a.cg, step_ch = blockDim.x - step_px * a.cg;
  px += (long long)img * a.pixels;
#pragma unroll 4
  for (; left > 0; --left) {
    use((size_t)px * a.cp + (size_t)g * a.cg + ch, (int)(g * a.cg) + ch);
    px += step_px;
    ch += step_ch;
    if (ch >= a.cg) {
      ch -= a.cg;
      ++px;
    }
  }
}
template <typename T> __global__ void group_norm_strided_stats_kernel(const GroupNormArgs a) {
  pdl_prologue();
  __shared__ float red[32];
  const T *in = (const T *)a.in;
  const unsigned lot = blockIdx.x / a.parts, part = blockIdx.x - lot * a.parts;
  const float count = (float)(min((part + 1) * a.part_values, (long long)a.pixels * a.cg) - part * a.part_values);
  float first = 0.0f, s = 0.0f, q = 0.0f, n = 0.0f;
  for_group_values<T>(a, [&](size_t at, int) {
    const float x = NormVec<T>::one(in[at]);
    if (n == 0.0f) first = x;
    n += 1.0f;
    s += x - first;
    q = fmaf(x - first, x - first, q);
  });
  const float mean = n > 0.0f ? s / n : 0.0f, m2 = fmaf(-s, mean, q), own = first + mean;
  const float all = block_sum(own * n, red) / count, d = own - all;
  const float sum = block_sum(n > 0.0f ? fmaf(d * n, d, m2 < 0.0f ? 0.0f : m2) : 0.0f, red);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = make_float2(all, sum);
}
template <typename T> __global__ void group_norm_strided_apply_kernel(const GroupNormArgs a) {
  typedef NormVec<T> V;
  pdl_prologue();
  __shared__ float red[32];
  const unsigned lot = blockIdx.x / a.parts, r = threadIdx.x; // a thread per part, of which there are no more than threads
  const float values = (float)((long long)a.pixels * a.cg);
  const float share = r < a.parts ? (float)(min((r + 1) * a.part_values, (long long)a.pixels * a.cg) - r * a.part_values) : 0.0f;
  const float2 o = r < a.parts ? a.partial[(size_t)lot * a.parts + r] : make_float2(0.0f, 0.0f);
  const float mean = block_sum(o.x * (share / values), red), d = o.x - mean;
  const float rstd = rsqrtf(block_sum(r < a.parts ? fmaf(d * d, share, o.y) : 0.0f, red) / values + a.eps);
  const T *in = (const T *)a.in;
  T *out = (T *)a.out;
  with_activation(a.act, [&](auto act) {
    for_group_values<T>(a, [&](size_t at, int ch) {
      const Pair v = both(fmaf((V::one(in[at]) - mean) * rstd, a.gamma[ch], a.beta[ch]));
      out[at] = V::back(activate<decltype(act)::value, V::kF32>(v).lo());
    });
  });
}

// To be called at load, on the device that will run it (conv_kernel_ready).
inline void group_norm_ready(const GroupNormPlan &p, bool f32) {
  if (p.form != NORM_SLAB || p.threads != kSlabThreads) return; // (small slabs stay below what a kernel has unasked)
  int device = 0;
  TPUCB_CUDA(cudaGetDevice(&device));
  auto set = [&](auto k) {
    static OncePerDevice ready; // one of each kernel
    ready.run(device, [] { TPUCB_CUDA(cudaFuncSetAttribute(decltype(k)::value, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)); });
  };
  if (f32 && p.aligned) set(KernelConstant<group_norm_slab_kernel<float, true, kSlabThreads>>());
  else if (f32) set(KernelConstant<group_norm_slab_kernel<float, false, kSlabThreads>>());
  else if (p.aligned) set(KernelConstant<group_norm_slab_kernel<uint16_t, true, kSlabThreads>>());
  else set(KernelConstant<group_norm_slab_kernel<uint16_t, false, kSlabThreads>>());
}
inline void launch_group_norm(const GroupNormArgs &a, const GroupNormPlan &p, bool f32, cudaStream_t s) {
  auto by_type = [&](auto type) {
    typedef decltype(type) T;
    auto rows = [&](auto nv, auto r, auto lanes) {
      constexpr int NV = decltype(nv)::value, R = decltype(r)::value, LANES = decltype(lanes)::value;
      if constexpr (NV * R <= 8 && (LANES != 8 || NV <= 2)) {
        if (a.cg == NV * NormVec<T>::N * (LANES ? LANES : (int)p.threads)) launch_k(group_norm_rows_kernel<T, NV, R, LANES, true>, p.grid, p.threads, 0, s, a);
        else launch_k(group_norm_rows_kernel<T, NV, R, LANES, false>, p.grid, p.threads, 0, s, a);
      }
    };
    auto by_rows = [&](auto nv, auto lanes) {
      if (p.rows == 2) rows(nv, std::integral_constant<int, 2>(), lanes);
      else rows(nv, std::integral_constant<int, 1>(), lanes);
    };
    auto by_nv = [&](auto use) {
      if (p.nv <= 1) use(std::integral_constant<int, 1>());
      else if (p.nv <= 2) use(std::integral_constant<int, 2>());
      else if (p.nv <= 4) use(std::integral_constant<int, 4>());
      else use(std::integral_constant<int, 8>());
    };
    switch (p.form) {
    case NORM_ROWS_WARP:
      if (p.lanes == 8) by_nv([&](auto nv) { by_rows(nv, std::integral_constant<int, 8>()); });
      else by_nv([&](auto nv) { by_rows(nv, std::integral_constant<int, 32>()); });
      break;
    case NORM_ROWS_BLOCK: by_nv([&](auto nv) { by_rows(nv, std::integral_constant<int, 0>()); }); break;
    case NORM_SLAB:
      if (p.threads == kSlabThreads) {
        if (p.aligned) launch_cluster_k(a.parts, group_norm_slab_kernel<T, true, kSlabThreads>, p.grid, p.threads, p.smem, s, a);
        else launch_cluster_k(a.parts, group_norm_slab_kernel<T, false, kSlabThreads>, p.grid, p.threads, p.smem, s, a);
      } else {
        if (p.aligned) launch_k(group_norm_slab_kernel<T, true, kSmallSlabThreads>, p.grid, p.threads, p.smem, s, a);
        else launch_k(group_norm_slab_kernel<T, false, kSmallSlabThreads>, p.grid, p.threads, p.smem, s, a);
      }
      break;
    case NORM_STREAMED: {
      auto both_passes = [&](auto aligned) {
        constexpr bool A = decltype(aligned)::value;
        launch_k(group_norm_stats_kernel<T, A>, p.grid, p.threads, p.smem, s, a);
        PdlConvScope overlap; // the second pass fetches gamma and beta while the first ends
        launch_k(group_norm_apply_kernel<T, A>, p.apply_grid, p.threads, (size_t)a.chunk_groups * sizeof(float2), s, a);
      };
      if (p.aligned) both_passes(std::true_type());
      else both_passes(std::false_type());
      break;
    }
    default:
      launch_k(group_norm_strided_stats_kernel<T>, p.grid, p.threads, 0, s, a);
      launch_k(group_norm_strided_apply_kernel<T>, p.grid, p.threads, 0, s, a);
    }
  };
  if (f32) by_type(float());
  else by_type(uint16_t());
}

} // namespace tpucb
