"""Where the sampler's weights end (tinybrain_b200/csrc/tb_sample_cut.h), on the CPU.

The weights' exponentials are built by adding to a double's exponent field, which
holds for exponents y = (x - max) / T down to about -708.  So no value at or above
the cut may lie more than 700 nats below the maximum, and none below it less, at
any size of the logits and the temperature.
"""
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinybrain_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "tb_sample_cut.h"
int main() {
    float top, T;
    while (scanf("%f %f", &top, &T) == 2) printf("%.9g\n", tb::lowest_weighted(top, T));
}
"""


@pytest.fixture(scope="module")
def cuts(tmp_path_factory):
    d = tmp_path_factory.mktemp("cut")
    (d / "cut.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", CSRC, "-o", str(d / "cut"), str(d / "cut.cpp")])

    def run(top, T):
        text = "\n".join(f"{float(a):.9g} {float(b):.9g}" for a, b in zip(top, T))
        r = subprocess.run([str(d / "cut")], input=text, capture_output=True, text=True, check=True)
        return np.array([np.float32(x) for x in r.stdout.split()], np.float32)

    return run


def test_no_value_above_the_cut_is_further_down_than_the_weights_reach(cuts):
    g = np.random.default_rng(0)
    n = 20000
    top = (g.choice([-1.0, 1.0], n) * 10.0 ** g.uniform(-30, 38, n)).astype(np.float32)
    T = np.where(g.random(n) < 0.5, np.abs(top.astype(np.float64)) * 10.0 ** g.uniform(-11, -5, n),  # 700 T about a step of top
                 10.0 ** g.uniform(-30, 30, n)).astype(np.float32)
    top[:4], T[:4] = [20.0, 3.3e7, 1e5, 0.0], [1e-8, 0.05, 1e-5, 1.0]
    keep = (T > 0) & np.isfinite(T) & np.isfinite(top)
    top, T = top[keep], T[keep]
    cut = cuts(top, T)
    below = np.nextafter(cut, np.float32(-np.inf))
    with np.errstate(over="ignore"):
        at, under = ((x.astype(np.float64) - top.astype(np.float64)) / T.astype(np.float64) for x in (cut, below))
    # (double's own rounding of max - 700 T: 2^-53 of max, less than 2^-28 of 700 T where cut and max differ)
    assert np.all(at >= -700.0 * (1 + 2.0 ** -27)) and np.all(cut <= top)
    assert np.all(under <= -700.0 * (1 - 2.0 ** -27))
    with np.errstate(over="ignore"):
        old = (top - np.float32(700.0) * T).astype(np.float32)
        far = (old.astype(np.float64) - top.astype(np.float64)) / T.astype(np.float64)
    assert (far < -708).any()  # rounded to nearest in 32 bits some lay beyond


def test_extreme_temperatures(cuts):
    big = np.finfo(np.float32).max
    cut = cuts([1.0, -5.0, 3e38, 1.0, 1.0], [1e-45, np.inf, 1e38, 3e38, np.inf])
    assert cut[0] == 1.0 and cut[1] == -np.inf and cut[4] == -np.inf
    assert cut[2] == -big and cut[3] == -big  # every finite value has a weight
