// What the module text says of a group_norm and of a fully_connected with activation or residual: arguments, checked before
// anything is built. Host only.
#pragma once
#include "module_text.h"

#include <cmath>
#include <cstring>
#include <functional>

namespace tpucb {

enum Activation { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4 };

inline int activation_from_string(const std::string &name, const std::string &op) {
  static const char *names[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};
  for (int i = 0; i < 5; ++i)
    if (name == names[i]) return i;
  throw Error(strfmt("%s: activation '%s' is none of none, relu, silu, gelu, gelu_tanh", op.c_str(), name.c_str()));
}

using WeightOf = std::function<const HostWeight &(const std::string &)>;

inline bool names_operand(const ParsedOp &op, size_t i) { return i < op.in.size() && op.in[i] != "-" && !op.in[i].empty(); }

// group_norm: operands input, gamma, beta ("-": ones, zeros); attributes groups, variance_epsilon (1e-5), activation (none).
struct GroupNormSpec {
  int groups = 1, act = ACT_NONE;
  float eps = 1e-5f;
  std::vector<float> gamma, beta; // with the channel pitch, zero behind the channels
};
inline GroupNormSpec group_norm_spec(const ParsedOp &op, const DevTensor &in, const DevTensor &out, const WeightOf &weight) {
  const char *nm = op.name.c_str();
  TPUCB_CHECK(in.dtype == out.dtype && out.dtype != 0, "group_norm %s: BF16 and fp32 are implemented, input and result of one type", nm);
  TPUCB_CHECK(in.n == out.n && in.c == out.c && in.h == out.h && in.w == out.w && in.cp == out.cp && !in.padded_rows() && !out.padded_rows(),
              "group_norm %s: input and result differ in shape", nm);
  TPUCB_CHECK(in.n > 0 && in.c > 0 && in.h > 0 && in.w > 0, "group_norm %s: empty tensor", nm);
  GroupNormSpec s;
  s.groups = op.geti("groups", 0);
  TPUCB_CHECK(s.groups > 0 && in.c % s.groups == 0, "group_norm %s: groups = %d does not divide the %d channels", nm, s.groups, in.c);
  s.eps = (float)op.getf("variance_epsilon", 1e-5);
  TPUCB_CHECK(s.eps > 0.0f && std::isfinite(s.eps), "group_norm %s: variance_epsilon must be a positive fp32 number", nm);
  s.act = activation_from_string(op.gets("activation", "none"), "group_norm " + op.name);
  TPUCB_CHECK((double)in.h * in.w < (double)(1 << 30) && (double)in.n * s.groups < 2147483648.0, "group_norm %s: too many pixels or groups", nm);
  auto affine = [&](size_t i, float absent) {
    std::vector<float> v(in.cp, 0.0f);
    std::fill(v.begin(), v.begin() + in.c, absent);
    if (names_operand(op, i)) {
      const auto &w = weight(op.in[i]).data;
      TPUCB_CHECK(w.size() == (size_t)in.c, "group_norm %s: operand %s has %zu values, expected %d", nm, op.in[i].c_str(), w.size(), in.c);
      std::copy(w.begin(), w.end(), v.begin());
    }
    return v;
  };
  s.gamma = affine(1, 1.0f);
  s.beta = affine(2, 0.0f);
  return s;
}

// The BF16 value that IEEE 754 rounds an fp32 one to (nearest even, infinities and NaN kept, overflow to infinity): weights of products whose
// results are rounded that way. (f32_to_bf16_bits makes the largest finite value of all that is not finite, whatever its sign.)
inline uint16_t bf16_bits_ieee(float v) {
  uint32_t u;
  std::memcpy(&u, &v, 4);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40u);
  return (uint16_t)((u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}

// fully_connected whose line names an activation or, as operand 7 behind the quantisation operands, a residual tensor.
inline bool linear_asked_for(const ParsedOp &op) { return op.attrs.count("activation") || names_operand(op, 7); }
struct LinearSpec {
  int m = 0, n = 0, act = ACT_NONE;
  int hw = 1;         // pixels of an input row: K is hw x channels
  int k_dev = 0;      // K on the device, with the input's channel pitch
  std::vector<float> bias; // zero behind the channels, for whole tiles of 256
  const HostWeight *filter = nullptr;
};
inline LinearSpec linear_spec(const ParsedOp &op, const DevTensor &in, const DevTensor &out, const DevTensor *res, const WeightOf &weight) {
  const char *nm = op.name.c_str();
  TPUCB_CHECK(in.dtype == out.dtype && out.dtype != 0, "fc %s: activation and residual need a BF16 or fp32 input and a result of its type", nm);
  LinearSpec s;
  s.act = activation_from_string(op.gets("activation", "none"), "fc " + op.name);
  if (op.geti("do_relu", 0)) {
    TPUCB_CHECK(!op.attrs.count("activation"), "fc %s: do_relu and activation exclude each other", nm);
    s.act = ACT_RELU;
  }
  TPUCB_CHECK(names_operand(op, 1), "fc %s: expects input, filter[, bias, -, -, -, -, residual]", nm);
  s.filter = &weight(op.in[1]);
  TPUCB_CHECK(s.filter->shape.size() <= 2, "fc %s: batched inner products have no activation or residual", nm);
  s.m = in.n;
  s.n = out.c;
  TPUCB_CHECK(in.n > 0 && in.c > 0 && in.h > 0 && in.w > 0 && out.c > 0, "fc %s: empty input or result", nm);
  TPUCB_CHECK((double)in.h * in.w * in.cp < (double)(1 << 29), "fc %s: input rows are too long", nm);
  TPUCB_CHECK(!in.padded_rows() && out.n == in.n && out.h == 1 && out.w == 1, "fc %s: output must be [m, n]", nm);
  s.hw = in.h * in.w;
  s.k_dev = s.hw * in.cp;
  const size_t k = (size_t)in.c * s.hw;
  TPUCB_CHECK(s.filter->data.size() == s.n * k, "fc %s: filter has %zu values, expected n*k = %zu", nm, s.filter->data.size(), s.n * k);
  s.bias.assign(round_up(out.cp, 256), 0.0f);
  if (names_operand(op, 2)) {
    const auto &b = weight(op.in[2]).data;
    TPUCB_CHECK(b.size() == (size_t)s.n, "fc %s: bias has %zu values, expected %d", nm, b.size(), s.n);
    std::copy(b.begin(), b.end(), s.bias.begin());
  }
  if (res)
    TPUCB_CHECK(res->dtype == out.dtype && res->n == out.n && res->c == out.c && res->h == 1 && res->w == 1 && res->cp == out.cp,
                "fc %s: residual %s must be [%d, %d] of the result's type", nm, op.in[7].c_str(), out.n, out.c);
  return s;
}

// ---- how a group norm runs (group_norm.cuh)
enum NormForm { NORM_ROWS_WARP = 0, NORM_ROWS_BLOCK, NORM_SLAB, NORM_STREAMED, NORM_STRIDED };
constexpr int kSlabThreads = 512, kSmallSlabThreads = 128, kStreamThreads = 256;
struct GroupNormPlan {
  int form = NORM_STRIDED;
  unsigned grid = 0, threads = 256;
  int nv = 1;             // vectors per thread
  int rows = 1;           // rows forms: rows at a time
  bool aligned = false;   // a vector's channels belong to one group
  int vecs = 1, lanes = 1, chunk_groups = 0, chunks = 0, parts = 1, part_pixels = 0;
  int col_split = 1, group_span = 32;
  int apply_parts = 1, apply_pixels = 0;
  unsigned apply_grid = 0;
  long long part_values = 0; // strided: of a group, per block
  size_t smem = 0;
};
// mode (option "norm_form"): 0 by size, else 1 + the form, where it can.
// Times in the comments are us per launch with three modules in flight / with one module's launches behind one another ("in a row").
inline GroupNormPlan group_norm_plan(int n, int pixels, int c, int groups, int es, int sm_count, int mode) {
  const int N = 16 / es, cg = c / groups;
  GroupNormPlan p;
  p.aligned = cg % N == 0;
  // strided: as many parts of a group as run at once, 2048 values or more each
  const long long values = (long long)pixels * cg, lots = (long long)n * groups;
  p.parts = (int)std::max(1LL, std::min({256LL, 8LL * sm_count / lots, values / 2048}));
  p.part_values = (values + p.parts - 1) / p.parts;
  p.parts = (int)((values + p.part_values - 1) / p.part_values);
  p.grid = (unsigned)(lots * p.parts);
  const GroupNormPlan strided = p;
  if (mode == 1 + NORM_STRIDED) return strided;
  if (pixels == 1 && (p.aligned || groups == 1) && mode <= 1 + NORM_ROWS_BLOCK) {
    // a thread keeps up to 8 vectors: 8 lanes of a warp, a warp, or a block, which is larger where there are too few rows for all SMs
    const int nvec = (cg + N - 1) / N;
    const bool many = n >= 8 * sm_count;
    auto units = [&](int lanes) { // of two neighbouring images where there are many, which share gamma and beta
      p.nv = 1;
      while (p.nv * lanes < nvec) p.nv *= 2;
      p.rows = many && p.nv <= 4 ? 2 : 1;
      return (long long)((n + p.rows - 1) / p.rows) * groups;
    };
    if (nvec <= 8 * 32 && mode != 1 + NORM_ROWS_BLOCK) {
      p.form = NORM_ROWS_WARP;
      p.parts = 1;
      p.threads = 128;
      p.lanes = nvec <= 16 ? 8 : 32;
      const int per_block = 128 / p.lanes;
      p.grid = (unsigned)((units(p.lanes) + per_block - 1) / per_block);
      return p;
    }
    if (nvec <= 8 * 512) {
      p.form = NORM_ROWS_BLOCK;
      p.parts = 1;
      const int want = many ? 4 : 2;
      p.threads = (unsigned)std::max(64, std::min(512, round_up((nvec + want - 1) / want, 32)));
      p.grid = (unsigned)units((int)p.threads);
      return p;
    }
  }
  // chunks: whole groups and whole vectors; the smallest such unit, or the whole row
  if (c >= 1 << 19 || lots * 8 >= 1LL << 31) return strided; // (small_div; the grid)
  int unit_groups = 1;
  while (unit_groups < groups && unit_groups * cg % N) ++unit_groups;
  const int unit_vecs = (unit_groups * cg + N - 1) / N;
  if (unit_vecs > kSlabThreads) return strided;
  const int units = (groups + unit_groups - 1) / unit_groups;
  auto lay_out = [&](int threads, int k, int parts) { // k units per chunk
    k = std::max(1, std::min({k, units, threads / unit_vecs, 256 / unit_groups})); // (256 groups: shared memory of norm_group_sums, 45 KB)
    p.vecs = k * unit_vecs;
    p.chunk_groups = std::min(groups, k * unit_groups);
    p.chunks = (groups + p.chunk_groups - 1) / p.chunk_groups;
    p.part_pixels = (pixels + parts - 1) / parts;
    p.parts = (pixels + p.part_pixels - 1) / p.part_pixels;
    const int per = p.aligned ? 1 : N;
    p.lanes = threads / p.vecs;
    p.nv = (p.part_pixels + p.lanes - 1) / p.lanes;
    p.threads = (unsigned)threads;
    p.grid = (unsigned)((long long)n * p.chunks * p.parts);
    // a column's pixel lanes are summed by several threads where there are few columns, eight lanes or more each
    const int group_width = p.aligned ? cg / N : cg;
    p.col_split = std::max(1, std::min(threads / (p.vecs * per), p.lanes / 8));
    p.group_span = round_up(p.col_split * group_width, 32);
    p.smem = ((size_t)threads * per + (size_t)p.chunk_groups * p.group_span / 32 * 33 + round_up(p.chunk_groups, 2)) * 4;
  };
  // Tensors whose passes take long enough that only their loops count: from 128 vectors per thread of the streamed form on.
  const bool large = (long long)n * pixels * ((c + N - 1) / N) >= 128LL * kStreamThreads * sm_count;
  // slab: 64 bytes of a pixel and more, in the shared memory of at most eight blocks; more of a pixel while two blocks per SM remain and one
  // block holds it (40 x 1280 x 16 x 16 by 80 bytes 24.9 / 28.7, by 320 10.6 / 18.5, streamed 19.1 / 32.8). Few
  // blocks per slab are best, for the sums of each cost the same: at most six where fewer hold it (2 x 320 x 96 x 96: by four 7.7 / 18.5, six
  // 9.0 / 16.4, eight 11.3 / 22.6, streamed 10.4 / 20.5). Where a block leaves no room for a second one on its SM, nothing fills the time of its loads
  // and sums: then only if they run at once, in clusters of up to six, on half of the SMs, else by more blocks (16 x 256 x 64 x 64 by two 17.8 /
  // 22.6, by three 16.3 / 22.3, streamed 18.8 / 28.5; 6 x 62 x 100 x 100 by seven 6.2 / 16.4, streamed 5.9 / 12.3; 2 x 320 x 128 x 128 by seven 17.5 /
  // 32.8, streamed 15.6 / 26.7). Large tensors only without clusters (100 x 640 x 32 x 32 70.5 / 80, streamed 70.5 / 97; by clusters of four
  // 48 x 320 x 64 x 64 82 / 92, streamed 65 / 83). A block of 128 threads where they have two vectors or fewer each (3000 x 64 x 3 x 3 9.9 / 14.4,
  // by 512 threads 35.6 / 39.0).
  int wide = (4 + unit_vecs - 1) / unit_vecs;
  while (2 * wide * unit_vecs <= kSlabThreads && (long long)n * ((units + 2 * wide - 1) / (2 * wide)) >= 2LL * sm_count &&
         (long long)pixels * 2 * wide * unit_vecs * 16 <= 90 * 1024)
    wide *= 2;
  lay_out(kSlabThreads, wide, 1);
  if (mode != 1 + NORM_STREAMED) {
    const size_t fixed = p.smem + (size_t)p.chunk_groups * 16, half = 113 * 1024;
    const long long slabs = (long long)n * p.chunks, lanes = p.lanes;
    auto parts_in = [&](size_t room) { // 9: none do
      const long long held = fixed < room ? (long long)((room - fixed) / (kSlabThreads * 16)) : 0;
      return held ? (int)std::min(9LL, (pixels + held * lanes - 1) / (held * lanes)) : 9;
    };
    auto try_slab = [&](int parts) {
      if (parts > 8 || (large && parts > 1 && mode == 0)) return false;
      lay_out(kSlabThreads, wide, parts);
      if (parts == 1 && p.vecs <= kSmallSlabThreads && pixels * p.vecs <= 2 * kSmallSlabThreads) {
        lay_out(kSmallSlabThreads, wide, 1);
        p.smem += (size_t)p.chunk_groups * 16 + (size_t)p.nv * kSmallSlabThreads * 16;
        p.form = NORM_SLAB;
        return true;
      }
      p.smem = fixed + (size_t)p.nv * kSlabThreads * 16;
      p.form = NORM_SLAB;
      return p.smem <= half || (p.parts <= 6 && slabs * p.parts <= sm_count && 2 * slabs * p.parts >= sm_count);
    };
    const int need = parts_in(2 * half);
    const long long spread = std::min({6LL, sm_count / slabs, (pixels + 2 * lanes - 1) / (2 * lanes)});
    if (try_slab((int)std::max<long long>(need, spread)) || try_slab(parts_in(half)) || (mode == 1 + NORM_SLAB && need <= 8)) return p;
  }
  if (unit_vecs > kStreamThreads) return strided;
  // streamed: chunks of whole rows where they fit, and as many parts of the image as run at once; a thread has 8 vectors at least
  const int most_units = std::max(1, 256 / unit_vecs);
  lay_out(kStreamThreads, most_units, 1);
  const long long slabs = (long long)n * p.chunks, per_part = 8LL * p.lanes;
  auto parts_of = [&](int blocks) { return (int)std::max(1LL, std::min((long long)blocks * sm_count / slabs, (pixels + per_part - 1) / per_part)); };
  // Blocks per SM of the two passes. Few leave fewer partial statistics and less around the loops, many hide the memory's latency; us in a row /
  // with three modules in flight, (1, 1), (1, 2), (2, 3): 4 x 128 x 128 x 128 24.6 / 10.7, 22.5 / 12.0, 20.5 / 13.8; 8 x 320 x 64 x 64
  // 28.7 / 14.1, 26.6 / 15.2, 22.6 / 16.5; 1 x 256 x 512 x 512 106 / 65, 91 / 71, 85 / 66; fp32 2 x 100 x 400 x 400 129 / 83, 116 / 83, 90 / 70.
  const int fs = large ? 2 : 1, fa = large ? 3 : 2;
  const int apply = parts_of(fa);
  lay_out(kStreamThreads, most_units, std::max(parts_of(fs), (int)((pixels + (1LL << 22) - 1) >> 22))); // (small_div)
  p.apply_pixels = (pixels + std::max(apply, p.parts) - 1) / std::max(apply, p.parts);
  p.apply_parts = (pixels + p.apply_pixels - 1) / p.apply_pixels;
  p.apply_grid = (unsigned)((long long)n * p.chunks * p.apply_parts);
  p.form = NORM_STREAMED;
  return p;
}

// ---- how an inner product runs on the tensor cores (linear_tc.cuh)
constexpr int kLinearMaxStages = 16;
constexpr int kLinearHeader = 1024;      // barriers
constexpr int kPairStaging = 16 * 2048;  // results on their way out, 32 rows x 32 channels per epilogue warp
struct LinearTcPlan {
  bool pair = false;  // two SMs per tile of 256 rows, persistent; else one of 128, and `split` CTAs share its K
  int nt = 0, split = 1, a_rows = 128, stages = 0, k_blocks = 0;
  unsigned tmem_cols = 512, grid = 0;
  size_t smem = 0;
};
// The sizes that follow from tiles of `nt` channels whose K is shared by `split` CTAs, or tiles of a pair.
inline LinearTcPlan linear_tc_sizes(bool pair, int nt, int split, int m, int k_dev, int n_pad, int sm_count) {
  LinearTcPlan l;
  l.pair = pair;
  l.nt = nt;
  l.k_blocks = (k_dev + 63) / 64;
  l.split = pair ? 1 : std::min(split, l.k_blocks);
  const long long n_tiles = (n_pad + nt - 1) / nt;
  if (pair) {
    const size_t stage = (size_t)(128 + nt / 2) * 128;
    const long long tiles = n_tiles * ((m + 255) / 256);
    l.stages = (int)std::min<size_t>(kLinearMaxStages, (227 * 1024 - kLinearHeader - kPairStaging - 1024) / stage);
    l.smem = 1024 + kLinearHeader + kPairStaging + l.stages * stage; // (more than half of an SM's: two pairs on the same SMs would wait for each other's tensor memory)
    l.grid = (unsigned)(2 * std::min<long long>(tiles, sm_count / 2));
    return l;
  }
  l.a_rows = std::min(128, round_up(m, 8));
  l.tmem_cols = 32;
  while ((int)l.tmem_cols < nt) l.tmem_cols *= 2;
  const size_t stage = (size_t)round_up(l.a_rows * 128, 1024) + (size_t)round_up(nt * 128, 1024);
  const int blocks = (l.k_blocks + l.split - 1) / l.split;
  // half of an SM's shared memory: two CTAs share it, one's epilogue beside the other's loop
  l.stages = std::max(1, (int)std::min<size_t>(std::min(blocks, kLinearMaxStages), (112 * 1024 - kLinearHeader - 1024) / stage));
  size_t ring = l.stages * stage;
  ring = std::max(ring, (l.stages - 1) * stage + 128 * 128);                                    // the tensor core reads 128 rows of the last stage
  if (l.split > 1) ring = std::max(ring, (size_t)nt * std::min(128, round_up(m, 32)) * 4); // the exchange of partial sums
  l.smem = 1024 + kLinearHeader + ring;
  l.grid = (unsigned)(n_tiles * ((m + 127) / 128) * l.split);
  return l;
}
// mode (option "linear_tiles"): 1 by size; 1000 * split + nt; 10000 + nt: pairs
// By size; us with three modules in flight / in a row:
//   Pairs where there are more tiles of 128 x 64 than SMs, and more than one of rows; 256 channels, 128 where those leave half of the
//   pairs idle. 256 x 4096 x 16384 31 / 37 (clusters of one 35 / 62), 8192 x 4096 x 4096 190 / 180 (222 / 240), 600 x 1000 x 5000 8.8 / 14.4 (8.8 /
//   18.3), 2048 x 512 x 2048 7.1 / 10.3 (6.7 / 12.3); 512 x 4096 x 4096 with 256 channels 14.0 / 26.8, with 128 15.6 / 18.6.
//   Else as many clusters as the SMs hold. Sharing K pays from about twelve K blocks per CTA on; below, and up to 64 CTAs, narrower tiles do:
//   256 x 1024 x 1024 with 32 channels 2.7 / 8.2, with 64 and two CTAs 4.0 / 10.2; 1 x 4096 x 4096 with 128 channels and four CTAs 6.2 / 12.3, with 64
//   and two 9.0 / 14.3, with 32 and one 7.0 / 16.4; 1 x 1024 x 1024 3.2 / 8.2. The exchange grows with the rows: 128 x 4096 x 4096 with 128 and
//   four 8.6 / 16.3, with 64 and two 8.1 / 14.3.
inline LinearTcPlan linear_tc_plan(int m, int k_dev, int n_pad, int sm_count, int mode) {
  if (mode >= 10000) return linear_tc_sizes(true, mode - 10000, 1, m, k_dev, n_pad, sm_count);
  if (mode >= 1000) return linear_tc_sizes(false, round_up(mode % 1000, 16), mode / 1000, m, k_dev, n_pad, sm_count);
  auto tiles = [&](int rows, int nt) { return (long long)((m + rows - 1) / rows) * ((n_pad + nt - 1) / nt); };
  if (m > 128 && tiles(128, 64) > sm_count) return linear_tc_sizes(true, tiles(256, 256) > sm_count / 4 ? 256 : 128, 1, m, k_dev, n_pad, sm_count);
  const int most = std::max(1, (k_dev + 63) / 64 / 12);
  int nt = m <= 32 ? 128 : 64, split;
  for (;; nt /= 2) {
    nt = std::min(nt, round_up(n_pad, 16));
    split = (int)std::max(1LL, std::min<long long>(std::min(8, most), sm_count / tiles(128, nt)));
    if (nt <= 16 || tiles(128, nt) * split >= 64) break;
  }
  return linear_tc_sizes(false, round_up(nt, 16), split, m, k_dev, n_pad, sm_count);
}
// ---- how an fp32 inner product runs (linear.cuh): 8 rm rows x 64 channels per tile, `split` blocks share its K
struct LinearF32Plan {
  int rm = 1, split = 1;
  unsigned grid = 0;
};
// mode (option "linear_tiles"): 1 by size; 1000 * split + rows of a tile, for fp32 8 to 56, rounded up to a multiple of 8
inline LinearF32Plan linear_f32_plan(int m, int k, int n_pad, int sm_count, int mode) {
  LinearF32Plan best;
  const int blocks = (k + 15) / 16;
  double least = 0;
  for (int rm = 1; rm <= 7; ++rm)
    for (int split = 1; split <= std::min(8, blocks); ++split) {
      if (mode >= 1000 && mode < 10000 && (rm != std::max(1, std::min(7, (mode % 1000 + 7) / 8)) || split != std::min(std::min(mode / 1000, 8), blocks))) continue;
      const long long grid = (long long)((n_pad + 63) / 64) * ((m + 8 * rm - 1) / (8 * rm)) * split;
      // Clocks of an SM, halfway between the busiest one's and the average. Per K block of 16 values a block takes about 96 rm of its multiply-adds
      // and what copies and barriers cost; alone on its SM it waits 2000 / stages for its copies and gets half of the multiply-adds' rate.
      const double ratio = (double)grid / sm_count, on_sm = 0.5 * (std::ceil(ratio) + std::max(1.0, ratio)), work = std::max(96.0 * rm + 150.0, 200.0);
      const double stages = std::min(8, 48 * 1024 / ((8 * rm + 64) * 80)), alone = std::max(2000.0 / stages, 2.0 * 96.0 * rm + 150.0);
      const double cost = (blocks + split - 1) / split * std::max(on_sm * work, alone) + on_sm * 500.0 + (split > 1 ? 1500.0 : 0.0);
      if (least != 0 && cost >= least) continue;
      least = cost;
      best.rm = rm;
      best.split = split;
      best.grid = (unsigned)grid;
    }
  return best;
}

} // namespace tpucb
