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


def shim(tmp_path):
    so = tmp_path / "libserving_shim.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", str(so),
                    os.path.join(HERE, "native", "serving_shim.cc")], check=True)
    return C.CDLL(str(so))


def test_every_exponential(tmp_path):
    L = shim(tmp_path)
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


def test_a_weight_is_told_without_a_division(tmp_path):
    """Terms on both sides of every boundary between two weights, and on it."""
    L = shim(tmp_path)
    rng = np.random.default_rng(3)
    term, total = [], []
    for bits in (32, 33, 34, 37, 41, 47, 62):
        s = [1 << bits, (1 << bits) + 1, (1 << bits) - 1 if bits > 32 else 1 << 32]
        s += [int(x) for x in rng.integers(1 << bits, 1 << bits + 1 if bits < 62 else (1 << 62) + 1, 5)]
        for x in s:
            for c in [1, 2, 3, 554, 555, 32767, 32768, 65535, 65536] + rng.integers(1, 65537, 60).tolist():
                at = (2 * c - 1) * x >> 17  # the weight is c - 1/2 here
                for t in range(at - 3, at + 5):
                    if 0 <= t <= 1 << 32:
                        term.append(t)
                        total.append(x)
    term.append(118945645)  # 554.49996, whose 32-bit estimate needs the exact answer
    total.append(14058110643)
    term, total = np.array(term, np.int64), np.array(total, np.uint64)
    want, agrees = np.zeros(len(term), np.int32), np.zeros(len(term), np.uint8)
    L.serving_weights(*(a.ctypes.data_as(C.c_void_p) for a in (term, total)), C.c_uint64(len(term)),
                      *(a.ctypes.data_as(C.c_void_p) for a in (want, agrees)))
    assert agrees.all() and want[-1] == 554
