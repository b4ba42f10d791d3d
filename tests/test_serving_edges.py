"""Edges of the serving operators that need no GPU: the score's arithmetic over
the whole 64-bit range, sizes at their bounds, what the wrappers take and
refuse."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def edges(tmp_path_factory):
    so = tmp_path_factory.mktemp("edges") / "libserving_edges.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", str(so),
                    os.path.join(HERE, "native", "serving_edges_shim.cc")], check=True)
    return C.CDLL(str(so))


def at(a):
    return a.ctypes.data_as(C.c_void_p)


@pytest.mark.parametrize("scale", [0, 1, 3, 268435456, 379625062, 1518500249, (1 << 31) - 1])
def test_scores_at_both_ends_of_the_sums(edges, scale):
    """Sums at the ends of int64, where a score passes 32 bits, at ties of both parities and anywhere."""
    rng = np.random.default_rng(scale)
    centers = [-(1 << 63), (1 << 63) - 1, 0, 1 << 47, -(1 << 47), 1 << 31, -(1 << 31), 1 << 62, -(1 << 62)]
    if scale:
        centers += [s * ((1 << 79) // scale) for s in (1, -1) if (1 << 79) // scale < 1 << 62]
    sums = [c + o for c in centers for o in list(range(-70000, 70001, 7)) + [s * (1 << b) + e for b in range(34)
            for s in (1, -1) for e in (-1, 0, 1)]]
    sums += [int(x) * 32768 for x in rng.integers(-1 << 33, 1 << 33, 20000)]  # ties
    sums += [int(x) for x in rng.integers(-1 << 63, (1 << 63) - 1, 200000)]
    sums = np.array([s for s in sums if -(1 << 63) <= s < 1 << 63], np.int64)
    got, want = np.zeros(len(sums), np.int32), np.zeros(len(sums), np.int32)
    edges.edge_scores(at(sums), C.c_uint64(len(sums)), C.c_uint32(scale), at(got), at(want))
    assert np.array_equal(got, want)


@pytest.fixture(scope="module")
def lib():
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib
    return _lib


@pytest.mark.parametrize("tokens,heads,kv_heads,d,window", [
    (1, 4, 1, 64, 0), (300, 4, 2, 128, 0), (300, 8, 1, 256, 96), (5000, 32, 8, 128, 0), (5000, 4, 2, 32, 17)])
def test_a_loose_bound_on_the_prompts_needs_no_more_scratch(lib, tokens, heads, kv_heads, d, window):
    """`longest` past the number of rows sizes the scratch as that number does, up to the last 32-bit one."""
    a = 1 << 20

    def need(longest):
        p = lib.PromptAttention(a, a, a, a, a, heads * d, kv_heads * d, kv_heads * d, heads * d, 3, tokens, longest,
                                heads, kv_heads, d, window, 1)
        return lib.lib().iris_prompt_attention_workspace(C.byref(p))

    rows = tokens + 15 if not window else min(tokens, window)
    assert need(tokens) >= rows * 4
    for longest in (tokens + 1, 1 << 31, 0xFFFFFF72, 0xFFFFFF80, 0xFFFFFFFF):
        assert need(longest) == need(tokens), longest


def test_a_place_that_was_not_found_is_read_inside_the_keys(edges):
    """A row whose maximum was never found (a wait that gave up) has the place 2^32 - 1."""
    for count in (1, 2, 127, 16256):
        for first in (0, 1, count - 1, count, 0xFFFFFFFF):
            got = edges.edge_place_within(C.c_uint32(first), C.c_uint32(count))
            assert got == (first if first < count else count - 1)
