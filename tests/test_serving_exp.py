"""The serving kernels' exponential on every distance it takes, as host code:
the 32-bit form equals softmax_exp_term, and the estimate that one bit corrects
is it or one less from its first distance on."""
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
    term, estimate, want = np.zeros(n, np.uint32), np.zeros(n, np.uint32), np.zeros(n, np.int64)
    L.serving_exp_terms(*(a.ctypes.data_as(C.c_void_p) for a in (term, estimate, want)))
    assert np.array_equal(term[1:].astype(np.int64), want[1:])
    below = L.serving_exact_below()
    off = want[below:] - estimate[below:].astype(np.int64)
    assert off.min() >= 0 and off.max() <= 1
    assert np.array_equal(ref.exp_term(np.arange(1, n)), want[1:])  # the tests' own restatement
