"""The serving kernels' exponential on every distance it takes, as host code:
the 32-bit form equals softmax_exp_term, and so does the estimate wherever it
has no doubt, which is nearly everywhere far from the maximum; the floor that
one bit corrects is it or one less from its first distance on."""
import ctypes as C
import os
import subprocess

import numpy as np

import serving_reference as ref

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_exponential(tmp_path):
    so = tmp_path / "libserving_shim.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", str(so),
                    os.path.join(HERE, "native", "serving_shim.cc")], check=True)
    L = C.CDLL(str(so))
    n = 1 << 20
    term, estimate, doubt, floor, want = (np.zeros(n, t) for t in (np.uint32, np.uint32, np.uint8, np.uint32, np.int64))
    L.serving_exp_terms(*(a.ctypes.data_as(C.c_void_p) for a in (term, estimate, doubt, floor, want)))
    assert np.array_equal(term[1:].astype(np.int64), want[1:])
    sure = doubt == 0
    sure[0] = False
    assert np.array_equal(estimate[sure].astype(np.int64), want[sure])
    assert doubt[1:].mean() < 0.25 and doubt[500000:].mean() < 0.01
    below = L.serving_exact_below()
    off = want[below:] - floor[below:].astype(np.int64)
    assert below % 32 == 0 and off.min() >= 0 and off.max() <= 1
    assert np.array_equal(ref.exp_term(np.arange(1, n)), want[1:])  # the tests' own restatement
