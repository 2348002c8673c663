"""The filter of a BF16 inner product with activation or residual is rounded as IEEE 754 has it."""
import os
import subprocess

import numpy as np
import pytest
import torch

import oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "norm_linear.h"
#include <iostream>
int main() {
  for (uint32_t u; std::cin.read((char *)&u, 4);) {
    float v;
    std::memcpy(&v, &u, 4);
    const uint16_t h = tpucb::bf16_bits_ieee(v);
    std::cout.write((const char *)&h, 2);
  }
}
"""


def test_rounding_against_torch(tmp_path):
    """Every upper half of a word with the lower halves where rounding decides."""
    src, exe = tmp_path / "t.cpp", str(tmp_path / "t")
    src.write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "tpu_compiler_b200", "csrc"), "-I", "/usr/local/cuda/include",
                    str(src), "-o", exe], check=True)
    low = np.array([0, 1, 0x7fff, 0x8000, 0x8001, 0xffff], np.uint32)
    u = (np.arange(1 << 16, dtype=np.uint32)[:, None] << 16 | low).reshape(-1)
    got = np.frombuffer(subprocess.run([exe], input=u.tobytes(), capture_output=True, check=True).stdout, np.uint16)
    want = torch.from_numpy(u.view(np.float32).copy()).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)
    nan = np.isnan(u.view(np.float32))
    assert np.array_equal(got[~nan], want[~nan])
    assert ((got[nan] & 0x7fff) > 0x7f80).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tiles", [1, 2032, 10064])
def test_weights_that_are_not_finite(tiles):
    """A weight of minus infinity, or one that rounds to it, keeps its sign; a NaN stays one."""
    from tpu_compiler_b200 import module
    rng = np.random.default_rng(3)
    m, k, n = 200, 72, 40
    x = O.bf16_round(rng.uniform(0.5, 1.0, (m, k)).astype(np.float32))
    f = rng.normal(0, 0.1, (n, k)).astype(np.float32)
    hard = [-np.inf, np.inf, np.nan, -3.4e38, 3.4e38, -3.39e38, 3.39e38, -1e38]
    f[:len(hard), 5] = hard
    mod = module(0)
    mod.set_option("linear_tiles", tiles)
    mod.load_text("input name=x shape=%d,%d dtype=BF16\nfully_connected name=y in=x,f shape=%d,%d dtype=BF16 activation=none\n" % (m, k, m, n), {"f": f})
    mod.set_tensor("x", x)
    mod.invoke()
    got = mod.get_tensor("y").astype(np.float64)
    mod.close()
    w = torch.from_numpy(f).to(torch.bfloat16).double().numpy()
    want = x.astype(np.float64) @ w.T
    infinite = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[infinite & ~np.isnan(want)], want[infinite & ~np.isnan(want)])
    # half a step of the result, and k sums, each rounded or cut to 24 bits
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -23 * k * (x.astype(np.float64) @ np.abs(w).T)
    assert (np.abs(got[~infinite] - want[~infinite]) <= tol[~infinite]).all()
