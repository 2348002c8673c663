"""The launches of inner products with activation or residual: every tile has its CTAs, in whole clusters; every K block of a tile has one of them."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLANS = r"""
#include "norm_linear.h"
#include <iostream>
using namespace tpucb;
#define EXPECT(x) do { if (!(x)) { std::cout << #x << " fails for " << what << std::endl; return 1; } } while (0)
// the K blocks of the CTAs of a tile, as the kernels divide them: none without one, all of them, each once
bool divides(int blocks, int split) {
  int at = 0;
  for (int r = 0; r < split; ++r) {
    const int from = (int)((long long)r * blocks / split), to = (int)((long long)(r + 1) * blocks / split);
    if (from != at || to <= from) return false;
    at = to;
  }
  return at == blocks;
}
int linear(int m, int k, int n, int sms, int mode) {
  std::stringstream ss;
  ss << "m " << m << " k " << k << " n " << n << " sms " << sms << " mode " << mode;
  const std::string what = ss.str();
  auto tiles = [&](long long pad, int rows, int channels) { return (pad + channels - 1) / channels * ((m + rows - 1) / rows); };
  {
    const int pad = round_up(n, 16), k_dev = round_up(k, 16);
    const LinearTcPlan l = linear_tc_plan(m, k_dev, pad, sms, mode);
    EXPECT(l.k_blocks == (k_dev + 63) / 64);
    EXPECT(l.pair == (mode >= 10000) || mode == 1);
    if (l.pair) {
      EXPECT(l.grid % 2 == 0 && l.grid >= 2 && l.grid <= 2 * tiles(pad, 256, l.nt) && (int)l.grid <= sms);
      EXPECT((long long)l.grid == std::min(2 * tiles(pad, 256, l.nt), (long long)sms / 2 * 2));
      EXPECT(l.smem > 114 * 1024); // one pair per two SMs: a second would wait for the first's tensor memory
    } else {
      EXPECT((long long)l.grid == tiles(pad, 128, l.nt) * l.split && l.grid % l.split == 0);
      EXPECT(divides(l.k_blocks, l.split));
    }
  }
  {
    const int pad = round_up(n, 4), k_dev = round_up(k, 4);
    const LinearF32Plan f = linear_f32_plan(m, k_dev, pad, sms, mode);
    EXPECT((long long)f.grid == tiles(pad, 8 * f.rm, 64) * f.split && f.grid % f.split == 0);
    EXPECT(f.split <= (k_dev + 15) / 16 && divides((k_dev + 15) / 16, f.split));
  }
  return 0;
}
int main() {
  for (int m : {1, 2, 8, 9, 17, 40, 128, 129, 200, 256, 257, 1000, 4100, 100000})
    for (int k : {1, 16, 17, 64, 65, 700, 768, 1000, 4096, 8192, 100000})
      for (int n : {1, 4, 5, 16, 17, 60, 250, 1000, 2050, 4096, 16384, 300000})
        for (int mode : {1, 1016, 1056, 2064, 8256, 8040, 3048, 5080, 10064, 10128, 10192, 10256})
          for (int sms : {148, 132, 20})
            if (linear(m, k, n, sms, mode)) return 1;
  std::cout << "sound" << std::endl;
}
"""


def test_grids_cover_the_tiles(tmp_path):
    src, exe = tmp_path / "t.cpp", str(tmp_path / "t")
    src.write_text(PLANS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "tpu_compiler_b200", "csrc"), "-I", "/usr/local/cuda/include",
                    str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True).stdout.strip() == "sound"
