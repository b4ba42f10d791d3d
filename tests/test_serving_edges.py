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


class Fake:
    """What the wrappers look at of a contiguous CUDA tensor, without one."""

    def __init__(self, *shape, dtype=None, device=0):
        import torch
        self.shape, self.dtype, self.index = shape, dtype or torch.int32, device
        self.is_cuda, self.device = True, f"cuda:{device}"

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def stride(self, axis=None):
        strides = [int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape))]
        return strides if axis is None else strides[axis]

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.index

    def data_ptr(self):
        return 1 << 20


def fakes(name):
    """A call's tensors, and the call."""
    import torch
    from iris_b200 import serving as S
    i64 = torch.int64
    return {
        "plan": (dict(held=Fake(2), fresh=Fake(2), table=Fake(2, 3), free_pages=Fake(4), parents=Fake(8)),
                 lambda t: S.page_plan(t["held"], t["fresh"], t["table"], t["free_pages"], 16, 8, parents=t["parents"])),
        "append": (dict(k=Fake(3, 64), v=Fake(3, 64), slots=Fake(3, dtype=i64), k_pages=Fake(2, 16, 64),
                        v_pages=Fake(2, 16, 64)), lambda t: S.page_append(*t.values())),
        "prompt": (dict(q=Fake(3, 64), k=Fake(3, 64), v=Fake(3, 64), offsets=Fake(2), out=Fake(3, 64)),
                   lambda t: S.prompt_attention(t["q"], t["k"], t["v"], t["offsets"], 3, heads=1, kv_heads=1,
                                                out=t["out"])),
        "tree": (dict(q=Fake(3, 64), k_pages=Fake(2, 16, 64), v_pages=Fake(2, 16, 64), table=Fake(1, 2), held=Fake(1),
                      offsets=Fake(2), masks=Fake(3, dtype=i64), positions=Fake(3), out=Fake(3, 64)),
                 lambda t: S.tree_attention(t["q"], t["k_pages"], t["v_pages"], t["table"], t["held"], t["offsets"],
                                            t["masks"], 3, 9, heads=1, kv_heads=1, positions=t["positions"],
                                            out=t["out"])),
        "accept": (dict(tokens=Fake(3), parents=Fake(3), picks=Fake(3), offsets=Fake(2), held=Fake(1), table=Fake(1, 2),
                        k_pages=Fake(2, 2, 16, 64), v_pages=Fake(2, 2, 16, 64)),
                   lambda t: S.tree_accept(t["tokens"], t["parents"], t["picks"], t["offsets"], t["held"], t["table"], 3,
                                           k_pages=t["k_pages"], v_pages=t["v_pages"])),
    }[name]


CALLS = ["plan", "append", "prompt", "tree", "accept"]


@pytest.mark.parametrize("call", CALLS)
def test_the_wrappers_refuse_tensors_of_two_devices(call):
    names = list(fakes(call)[0])
    for name in names[1:]:
        tensors, run = fakes(call)
        tensors[name].index = 1
        with pytest.raises(ValueError, match=f"^{name}: "):
            run(tensors)


@pytest.mark.parametrize("call,name", [
    ("prompt", "longest"), ("prompt", "heads"), ("prompt", "kv_heads"), ("prompt", "window"), ("prompt", "scale_q32"),
    ("tree", "nodes"), ("tree", "longest"), ("tree", "heads"), ("tree", "kv_heads"), ("tree", "window"),
    ("tree", "scale_q32"), ("plan", "page_size"), ("plan", "tokens"), ("accept", "path_width")])
def test_the_wrappers_refuse_numbers_that_are_no_32_bit_counts(call, name):
    """Numbers past 32 bits, and negative ones, are not cut to some other count."""
    from iris_b200 import serving as S
    t, _ = fakes(call)
    numbers = dict(prompt=dict(longest=3, heads=1, kv_heads=1, window=0, scale_q32=0),
                   tree=dict(nodes=3, longest=9, heads=1, kv_heads=1, window=0, scale_q32=0),
                   plan=dict(page_size=16, tokens=8), accept=dict(path_width=3))[call]
    for bad in (-1, 1 << 32, (1 << 32) + numbers[name], -(1 << 40)):
        with pytest.raises(ValueError, match=f"^{name}: .*2\\^32"):
            run = dict(prompt=S.prompt_attention, tree=S.tree_attention, plan=S.page_plan, accept=S.tree_accept)[call]
            run(**t, **{**numbers, name: bad})


def test_offsets_have_an_end():
    from iris_b200 import serving as S
    t, _ = fakes("prompt")
    t["offsets"] = Fake(0)
    with pytest.raises(ValueError, match="^requests: -1"):
        S.prompt_attention(**t, longest=3, heads=1, kv_heads=1)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("shape", [(), (3,), (1, 2), (1, 2, 16, 64), (0,)])
def test_the_wrappers_name_the_tensor_of_a_wrong_shape(call, shape):
    """A tensor with other axes than the call's is refused by its name, whatever they are."""
    for name, x in fakes(call)[0].items():
        if len(shape) == len(x.shape):
            continue
        tensors, run = fakes(call)
        tensors[name] = Fake(*shape, dtype=x.dtype)
        with pytest.raises(ValueError, match=name):
            run(tensors)


def test_trees_past_a_grid_of_segments_need_no_scratch(lib):
    """Bounds past 65,535 segments of 1,024 keys are the row kernel's."""
    a = 1 << 20

    def need(longest):
        t = lib.TreeAttention(a, a, a, a, a, a, a, None, a, 128, 128, 8, 1, 2, 1 << 23, 16, 2, longest, 2, 1, 64, 0, 1)
        return lib.lib().iris_tree_attention_workspace(C.byref(t))

    assert need(65535 * 1024) >= 65535 * 1024 * 16
    for longest in (65535 * 1024 + 1, 1 << 27):
        assert need(longest) == 0
