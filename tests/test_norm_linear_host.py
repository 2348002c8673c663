"""group_norm and fully_connected with activation / residual, what needs no GPU: the checks of the arguments (compiled for the host)
and the oracle's definitions against torch's."""
import os
import subprocess

import numpy as np
import pytest
import torch

import oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHECKS = r"""
#include "norm_linear.h"
#include <iostream>
using namespace tpucb;
// stdin: weight lines "w name d0,d1,..", then op lines; the results of input ops are their operands. stdout: a line per other op.
int main() {
  std::map<std::string, HostWeight> weights;
  std::map<std::string, DevTensor> tensors;
  for (std::string line; std::getline(std::cin, line);) {
    if (line.rfind("w ", 0) == 0) {
      std::stringstream ss(line.substr(2));
      std::string name, dims;
      ss >> name >> dims;
      HostWeight w;
      size_t n = 1;
      for (auto &d : split(dims, ',')) { w.shape.push_back(atoll(d.c_str())); n *= w.shape.back(); }
      w.data.assign(n, 0.5f);
      weights[name] = w;
      continue;
    }
    const ParsedOp op = parse_line(line);
    DevTensor t;
    t.dtype = op.dtype == "INT8" ? 0 : (op.dtype == "BF16" ? 1 : 2);
    int64_t d[4] = {1, 1, 1, 1};
    for (size_t i = 0; i < op.shape.size(); ++i) d[i] = op.shape[i];
    t.n = d[0]; t.c = d[1]; t.h = d[2]; t.w = t.wphys = d[3];
    t.cp = round_up(t.c, t.dtype == 2 ? 4 : 16);
    if (op.type == "input") { tensors[op.name] = t; continue; }
    auto weight = [&](const std::string &nm) -> const HostWeight & {
      TPUCB_CHECK(weights.count(nm), "weight '%s' was not registered", nm.c_str());
      return weights[nm];
    };
    try {
      if (op.type == "group_norm") {
        const GroupNormSpec s = group_norm_spec(op, tensors.at(op.in[0]), t, weight);
        std::cout << "ok groups=" << s.groups << " act=" << s.act << " eps=" << s.eps << " gamma0=" << s.gamma[0] << " gammas=" << s.gamma.size() << std::endl;
      } else if (!linear_asked_for(op)) {
        std::cout << "plain" << std::endl;
      } else {
        const DevTensor *res = names_operand(op, 7) ? &tensors.at(op.in[7]) : nullptr;
        const LinearSpec s = linear_spec(op, tensors.at(op.in[0]), t, res, weight);
        std::cout << "ok m=" << s.m << " n=" << s.n << " k=" << s.k_dev << " act=" << s.act << " bias0=" << s.bias[0] << std::endl;
      }
    } catch (const Error &e) {
      std::cout << "refused: " << e.what() << std::endl;
    }
  }
}
"""


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("checks")
    src, exe = d / "t.cpp", str(d / "t")
    src.write_text(CHECKS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "tpu_compiler_b200", "csrc"), "-I", "/usr/local/cuda/include",
                    str(src), "-o", exe], check=True)

    def run(lines):
        return subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True).stdout.splitlines()
    return run


NORM_IN = ["w g 48", "w b 48", "w short 47", "input name=x shape=2,48,5,3 dtype=BF16", "input name=q shape=2,48,5,3 dtype=INT8",
           "input name=none shape=0,48 dtype=BF16", "input name=wide shape=1,1,32768,32768 dtype=BF16"]


@pytest.mark.parametrize("line,answer", [
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 activation=silu variance_epsilon=1e-6",
     "ok groups=4 act=2 eps=1e-06 gamma0=0.5 gammas=48"),
    ("group_norm name=y in=x,-,- shape=2,48,5,3 dtype=BF16 groups=48", "ok groups=48 act=0 eps=1e-05 gamma0=1 gammas=48"),
    ("group_norm name=y in=x shape=2,48,5,3 dtype=BF16 groups=1 activation=gelu", "ok groups=1 act=3 eps=1e-05 gamma0=1 gammas=48"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16", "does not divide"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=5", "does not divide"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=-4", "does not divide"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=FP32 groups=4", "one type"),
    ("group_norm name=y in=q,g,b shape=2,48,5,3 dtype=INT8 groups=4", "BF16 and fp32 are implemented"),
    ("group_norm name=y in=x,g,b shape=2,48,5,4 dtype=BF16 groups=4", "differ in shape"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 activation=mish", "is none of"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 variance_epsilon=0", "must be a positive"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 variance_epsilon=-1e-5", "must be a positive"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 variance_epsilon=nan", "must be a positive"),
    ("group_norm name=y in=x,g,b shape=2,48,5,3 dtype=BF16 groups=4 variance_epsilon=1e-60", "must be a positive"),
    ("group_norm name=y in=x,short,b shape=2,48,5,3 dtype=BF16 groups=4", "47 values, expected 48"),
    ("group_norm name=y in=x,g,lost shape=2,48,5,3 dtype=BF16 groups=4", "was not registered"),
    ("group_norm name=y in=none,-,- shape=0,48 dtype=BF16 groups=4", "empty tensor"),
    ("group_norm name=y in=wide shape=1,1,32768,32768 dtype=BF16 groups=1", "too many pixels"),
])
def test_group_norm_arguments(checks, line, answer):
    got, = checks(NORM_IN + [line])
    assert answer in got and got.startswith("ok" if answer.startswith("ok") else "refused"), got


LINEAR_IN = ["w f 20,48", "w img 20,720", "w batched 2,20,48", "w b 20", "w b19 19", "input name=x shape=3,48 dtype=BF16",
             "input name=xi shape=3,48,5,3 dtype=BF16", "input name=x32 shape=3,40 dtype=FP32", "w f32 20,40", "input name=q shape=3,48 dtype=INT8",
             "input name=r shape=3,20 dtype=BF16", "input name=rbad shape=4,20 dtype=BF16", "input name=r32 shape=3,20 dtype=FP32",
             "input name=none shape=0,48 dtype=BF16", "input name=long shape=1,16,20000,20000 dtype=BF16"]


@pytest.mark.parametrize("line,answer", [
    ("fully_connected name=y in=x,f,b shape=3,20 dtype=BF16", "plain"),
    ("fully_connected name=y in=x,f,b,-,-,-,-,- shape=3,20 dtype=BF16 do_relu=1", "plain"),
    ("fully_connected name=y in=x,f,b shape=3,20 dtype=BF16 activation=none", "ok m=3 n=20 k=48 act=0 bias0=0.5"),
    ("fully_connected name=y in=x,f shape=3,20 dtype=BF16 activation=gelu_tanh", "ok m=3 n=20 k=48 act=4 bias0=0"),
    ("fully_connected name=y in=x,f,-,-,-,-,-,r shape=3,20 dtype=BF16 do_relu=1", "ok m=3 n=20 k=48 act=1 bias0=0"),
    ("fully_connected name=y in=xi,img,b shape=3,20 dtype=BF16 activation=silu", "ok m=3 n=20 k=720 act=2 bias0=0.5"),
    ("fully_connected name=y in=x32,f32,b,-,-,-,-,r32 shape=3,20 dtype=FP32", "ok m=3 n=20 k=40 act=0 bias0=0.5"),
    ("fully_connected name=y in=x,f,b shape=3,20 dtype=BF16 activation=swish", "is none of"),
    ("fully_connected name=y in=x,f,b shape=3,20 dtype=BF16 activation=relu do_relu=1", "exclude each other"),
    ("fully_connected name=y in=q,f,b shape=3,20 dtype=INT8 activation=relu", "need a BF16 or fp32"),
    ("fully_connected name=y in=x,f,b shape=3,20 dtype=FP32 activation=relu", "need a BF16 or fp32"),
    ("fully_connected name=y in=x,batched,b shape=3,20 dtype=BF16 activation=relu", "batched"),
    ("fully_connected name=y in=x,f,b shape=3,21 dtype=BF16 activation=relu", "filter has 960 values, expected n*k = 1008"),
    ("fully_connected name=y in=x,f,b19 shape=3,20 dtype=BF16 activation=relu", "bias has 19 values"),
    ("fully_connected name=y in=x,f,lost shape=3,20 dtype=BF16 activation=relu", "was not registered"),
    ("fully_connected name=y in=x,f,b shape=2,20 dtype=BF16 activation=relu", r"output must be [m, n]"),
    ("fully_connected name=y in=x,f,b shape=3,20,1,2 dtype=BF16 activation=relu", r"output must be [m, n]"),
    ("fully_connected name=y in=x,f,b,-,-,-,-,rbad shape=3,20 dtype=BF16", "residual rbad must be"),
    ("fully_connected name=y in=x,f,b,-,-,-,-,r32 shape=3,20 dtype=BF16", "residual r32 must be"),
    ("fully_connected name=y in=none,f,b shape=0,20 dtype=BF16 activation=relu", "empty"),
    ("fully_connected name=y in=long,f,b shape=1,20 dtype=BF16 activation=relu", "too long"),
    ("fully_connected name=y in=x shape=3,20 dtype=BF16 activation=relu", "expects input, filter"),
])
def test_linear_arguments(checks, line, answer):
    got, = checks(LINEAR_IN + [line])
    assert answer in got and (got.startswith("refused") or answer.startswith(("ok", "plain"))), got


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_oracle_definitions_against_torch(act):
    """2^-45: some hundred roundings of 2^-53 each."""
    f = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act]
    rng = np.random.default_rng(3)
    x, g, b = rng.normal(1, 2, (2, 12, 5, 3)), rng.normal(1, 0.2, 12), rng.normal(0, 0.2, 12)
    eps = float(np.float32(1e-3))
    for groups in (1, 3, 12):
        want = f(torch.nn.functional.group_norm(torch.tensor(x), groups, torch.tensor(g), torch.tensor(b), eps)).numpy()
        assert np.abs(O.group_norm64(x, groups, g, b, 1e-3, act) - want).max() < 2 ** -45 * 16
    rows = x.reshape(24, 15)
    want = f(torch.nn.functional.layer_norm(torch.tensor(rows), (15,), None, None, eps)).numpy()
    assert np.abs(O.group_norm64(rows, 1, None, None, 1e-3, act) - want).max() < 2 ** -45 * 16
    w, bias, r = rng.normal(0, 1, (7, 15)), rng.normal(0, 1, 7), rng.normal(0, 1, (24, 7))
    want = (f(torch.tensor(rows) @ torch.tensor(w).T + torch.tensor(bias)) + torch.tensor(r)).numpy()
    assert np.abs(O.linear64(rows, w, bias, act, r) - want).max() < 2 ** -45 * 64


@pytest.mark.parametrize("line", ["group_norm name=y in=x shape=2,16 dtype=FP32 groups=1",
                                  "fully_connected name=y in=x,f,b shape=2,16 dtype=FP32 activation=gelu",
                                  "fully_connected name=y in=x,f,b,-,-,-,-,x shape=2,16 dtype=FP32"])
def test_int8_quantisation_refuses(line):
    """Neither op has an INT8 form: an fp32 graph with one is not quantised into one without it."""
    from tpu_compiler_b200 import quantize
    weights = {"f": np.ones((16, 16), np.float32), "b": np.ones(16, np.float32)}
    with pytest.raises(NotImplementedError, match="is not covered"):
        quantize.quantize_module("input name=x shape=2,16 dtype=FP32\n" + line + "\n", weights, {"x": 1.0, "y": 2.0})


PLANS = r"""
#include "norm_linear.h"
#include <iostream>
using namespace tpucb;
#define EXPECT(x) do { if (!(x)) { std::cout << #x << " fails for " << what << std::endl; return 1; } } while (0)
int norm(int n, int pixels, int c, int groups, int es, int sms, int mode) {
  std::stringstream ss;
  ss << "n " << n << " pixels " << pixels << " c " << c << " groups " << groups << " es " << es << " sms " << sms << " mode " << mode;
  const std::string what = ss.str();
  const GroupNormPlan p = group_norm_plan(n, pixels, c, groups, es, sms, mode);
  const int N = 16 / es, cg = c / groups, nvec = (cg + N - 1) / N;
  if (p.form == NORM_ROWS_WARP || p.form == NORM_ROWS_BLOCK) {
    const bool warp = p.form == NORM_ROWS_WARP;
    const int lanes = warp ? p.lanes : (int)p.threads;
    EXPECT(pixels == 1 && (cg % N == 0 || groups == 1));
    EXPECT(p.nv <= 8 && p.nv * lanes >= nvec && (p.nv == 1 || p.nv / 2 * lanes < nvec));
    EXPECT((long long)p.grid * (warp ? p.threads / p.lanes : 1) >= (long long)((n + p.rows - 1) / p.rows) * groups);
    EXPECT(p.threads % 32 == 0 && p.threads <= 512 && (p.rows == 1 || p.nv <= 4));
  } else if (p.form == NORM_SLAB || p.form == NORM_STREAMED) {
    const bool slab = p.form == NORM_SLAB;
    EXPECT(slab ? p.threads == kSlabThreads || (p.threads == kSmallSlabThreads && p.parts == 1 && p.smem <= 48 * 1024) : p.threads == kStreamThreads);
    EXPECT(p.chunk_groups >= 1 && p.chunk_groups <= 256 && (long long)p.chunks * p.chunk_groups >= groups);
    EXPECT((p.chunks - 1) * p.chunk_groups < groups);
    EXPECT((long long)p.vecs * N >= (long long)p.chunk_groups * cg && (p.chunks == 1 || p.chunk_groups * cg == p.vecs * N));
    EXPECT(p.lanes >= 1 && p.vecs * p.lanes <= (int)p.threads && p.nv * p.lanes >= p.part_pixels && p.col_split >= 1);
    EXPECT((long long)p.parts * p.part_pixels >= pixels && (long long)(p.parts - 1) * p.part_pixels < pixels);
    EXPECT(p.grid == (unsigned)(n * p.chunks * p.parts) && (long long)n * p.chunks * p.parts < 1LL << 31 && p.part_pixels <= 1 << 22);
    const int per = p.aligned ? 1 : N, group_width = p.aligned ? cg / N : cg;
    EXPECT(p.group_span % 32 == 0 && p.group_span >= p.col_split * group_width);
    const size_t tab = ((size_t)p.threads * per + (size_t)p.chunk_groups * (p.group_span + p.group_span / 32)) * 4;
    if (slab) {
      EXPECT(p.parts <= 8 && p.smem <= 227 * 1024);
      EXPECT(p.smem >= tab + (size_t)p.nv * p.threads * 16 + (size_t)p.chunk_groups * 16);
    } else {
      EXPECT(p.smem <= 48 * 1024 && p.smem >= tab + (size_t)p.chunk_groups * 4 && p.smem >= (size_t)p.chunk_groups * 8);
      EXPECT((long long)p.apply_parts * p.apply_pixels >= pixels && (long long)(p.apply_parts - 1) * p.apply_pixels < pixels);
      EXPECT(p.apply_grid == (unsigned)(n * p.chunks * p.apply_parts) && p.apply_pixels <= 1 << 22);
    }
  } else {
    EXPECT(p.parts <= (int)p.threads && p.grid == (unsigned)(n * groups * p.parts) && (long long)n * groups * p.parts < 1LL << 31);
    EXPECT(p.part_values * p.parts >= (long long)pixels * cg && p.part_values * (p.parts - 1) < (long long)pixels * cg);
  }
  return 0;
}
int linear(int m, int k, int n, int sms, int mode) {
  std::stringstream ss;
  ss << "m " << m << " k " << k << " n " << n << " sms " << sms << " mode " << mode;
  const std::string what = ss.str();
  const int n_pad = round_up(n, 16);
  const LinearTcPlan l = linear_tc_plan(m, k, n_pad, sms, mode);
  EXPECT(l.nt >= 16 && l.nt <= 256 && l.nt % (l.pair ? 64 : 16) == 0 && l.split >= 1 && l.split <= 8);
  EXPECT(l.split <= (k + 63) / 64 && (l.pair ? l.split == 1 : true));
  EXPECT(l.smem <= 227 * 1024 && l.stages <= kLinearMaxStages && l.stages >= std::min(2, (l.k_blocks + l.split - 1) / l.split));
  EXPECT((l.tmem_cols & (l.tmem_cols - 1)) == 0 && l.tmem_cols >= 32 && l.tmem_cols <= 512 && (int)l.tmem_cols >= l.nt * (l.pair ? 2 : 1));
  EXPECT(l.pair || (l.a_rows >= std::min(m, 128) && l.a_rows <= 128 && l.a_rows % 8 == 0));
  const LinearF32Plan f = linear_f32_plan(m, k, n, sms, mode);
  EXPECT(f.rm >= 1 && f.rm <= 7 && f.split >= 1 && f.split <= 8);
  return 0;
}
int main() {
  const int channels[] = {1, 3, 7, 8, 16, 33, 62, 64, 100, 320, 512, 1025, 2048, 4100, 8192, 20000, 524287, 600000};
  const int pixels[] = {1, 2, 9, 64, 1767, 4096, 10000, 90000, 262144, 50000000};
  for (int c : channels)
    for (int g = 1; g <= c; g = g < 64 ? g + 1 : g * 2)
      for (int px : pixels)
        for (int n : {1, 2, 9, 300, 8192})
          for (int es : {2, 4})
            for (int mode = 0; mode <= 5; ++mode)
              for (int sms : {148, 20})
                if (c % g == 0 && (long long)c * px * n < 1LL << 36 && (long long)n * g < 1LL << 31 && norm(n, px, c, g, es, sms, mode)) return 1;
  for (int c : {512, 2048, 8192, 524287, 524286})
    for (int es : {2, 4})
      for (int mode = 0; mode <= 5; ++mode)
        if (norm(3, 12000, c, c, es, 148, mode)) return 1;
  for (int m : {1, 2, 17, 128, 129, 200, 256, 1000, 4100, 100000})
    for (int k : {1, 16, 64, 700, 768, 1000, 4096, 8192, 100000})
      for (int n : {1, 16, 17, 60, 250, 1000, 2050, 4096, 16384, 300000})
        for (int mode : {1, 1016, 2064, 8256, 3048, 5080, 10064, 10128, 10192, 10256})
          for (int sms : {148, 20})
            if (linear(m, k, n, sms, mode)) return 1;
  std::cout << "sound" << std::endl;
}
"""


def test_plans_cover_their_tensors_within_the_limits(tmp_path):
    """Every pixel, channel and group has a block, shared and tensor memory suffice, grids stay within what a launch may have."""
    src, exe = tmp_path / "t.cpp", str(tmp_path / "t")
    src.write_text(PLANS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "tpu_compiler_b200", "csrc"), "-I", "/usr/local/cuda/include",
                    str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True).stdout.strip() == "sound"
