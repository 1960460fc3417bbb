"""Numerics of the verification kernels that need no GPU: the 64-bit exponential of the sweeps over a row, compiled
for the host from the kernels' own header and compared with ``expl`` in 80 bits."""

from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "mlx-motif_b200" / "csrc"

HARNESS = r"""
#include "sweep.cuh"
// weight and exp((l - m) / tau) with its exponent in 80 bits; the weight's relative error
extern "C" void run(const float* l, const float* m, int n, double tau, double* w, double* y, double* err) {
  double table[motif::kSweepTable];
  for (int j = 0; j < motif::kSweepTable; ++j) table[j] = exp2l((long double)j / motif::kSweepTable);
  const double k = 1.0 / tau * 1.4426950408889634074;
  for (int i = 0; i < n; ++i) {
    w[i] = motif::sweep_weight(l[i], (double)m[i], k, table);
    const long double x = ((long double)l[i] - (long double)m[i]) / tau, e = expl(x);
    y[i] = (double)(x * 1.4426950408889634073599L);
    err[i] = e > 0 ? (double)(fabsl((long double)w[i] - e) / e) : (w[i] != 0.0);
  }
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    d = tmp_path_factory.mktemp("sweep")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run([gxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-ffp-contract=off", "-I", str(CSRC), "-o", str(d / "h.so"),
                    str(d / "h.cpp")], check=True)
    f = C.CDLL(str(d / "h.so")).run

    def call(l, m, tau):
        l, m = (np.ascontiguousarray(np.broadcast_to(np.asarray(x, np.float32), np.shape(l))) for x in (l, m))
        out = [np.empty(l.size) for _ in range(3)]
        f(*(x.ctypes.data_as(C.c_void_p) for x in (l, m)), l.size, C.c_double(tau),
          *(o.ctypes.data_as(C.c_void_p) for o in out))
        return out

    return call


@pytest.mark.parametrize("tau", [1e-6, 0.3, 0.5, 0.7, 1.0, 1.3, 50.0, 1e6])
def test_sweep_weight_is_exp(run, tau):
    """Within (2.8·|y| + 3)·2^-53, the bound of its comment, down to 2^-1021; at most 1; 0 below 2^-1023."""
    rng = np.random.default_rng(1)
    n = 200000
    for size in (1.0, 50.0, 1e4, 1e20):  # of the maximum
        m = (rng.standard_normal(n) * size).astype(np.float32)
        span = -rng.random(n) * rng.choice([1e-3, 1.0, 60.0, 1100.0], n) * tau * np.log(2)
        l = np.minimum((m + span).astype(np.float32), m)
        w, y, err = run(l, m, tau)
        assert (w <= 1.0).all() and (w >= 0.0).all() and (w[l == m] == 1.0).all()
        live = y > -1021
        assert (err[live] <= (2.8 * np.abs(y[live]) + 3) * 2.0**-53).all()
        assert (w[y < -1023] == 0).all()


def test_sweep_weight_of_extreme_logits(run):
    """Rows of one very large value (its weight is 1), and entries as far below the maximum as the type goes."""
    top = np.finfo(np.float32).max
    for tau in (1e-6, 0.3, 0.7, 1.0, 1e6):
        for v in (top, -top, 1e20, -1e20, 3e38, -65504.0):
            w, _, _ = run(np.full(4, v), v, tau)
            assert (w == 1.0).all(), (v, tau, w)
        w, _, _ = run(np.array([-top, -1e20, -np.inf, np.nextafter(np.float32(1e20), np.float32(0))]), 1e20, tau)
        assert (w == 0.0).all()
        w, _, _ = run(np.array([-top, -np.inf]), top, tau)
        assert (w == 0.0).all()
