"""The serving operators' arithmetic against the oracle's: the plain restatement
that the GPU tests compare with (tests/serving_reference.py), and the kernels
themselves, give the scores, the softmax and the value sums of the oracle
(mistral.rs:130-145, ops.rs:233-276, tensor.rs:530-536)."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as ref

I32P = C.POINTER(C.c_int32)


@pytest.fixture(scope="module")
def O():
    from oracle import oracle
    oracle.build()
    return oracle.lib()


def at(a):
    return a.ctypes.data_as(I32P)


def rows(rng, shape, kind):
    if kind == "full":
        x = rng.integers(-2**31, 2**31, shape)
        return np.where(rng.random(shape) < 0.2, np.where(rng.random(shape) < 0.5, -2**31, 2**31 - 1), x).astype(np.int32)
    x = rng.normal(size=shape) * 1.2
    if kind == "wide":
        x = np.where(rng.random(shape) < 0.05, x * 300, x)
    return (x * 65536).astype(np.int32)


def score(O, q, k, scale):
    return O.oracle_scaled_score(at(q), at(k), q.size, scale) if scale else O.oracle_dot_bits(at(q), at(k), q.size)


def softmax(O, scores):
    out = np.zeros(scores.size, np.int32)
    O.oracle_attention_softmax(at(scores), scores.size, at(out))
    return out


def attend(O, q, k, v, scale):
    """One query over its keys, by the oracle's functions."""
    q, k, v = (np.ascontiguousarray(x) for x in (q, k, v))
    w = softmax(O, np.array([score(O, q, x, scale) for x in k], np.int32))
    out = np.zeros(q.size, np.int32)
    for d in range(q.size):
        acc = 0
        for t in range(len(k)):
            acc = O.oracle_mac_bits(acc, int(w[t]), int(v[t, d]))
        out[d] = O.oracle_requantize(acc)
    return out


@pytest.mark.parametrize("kind", ["model", "wide", "full"])
@pytest.mark.parametrize("d,scaled", [(4, True), (64, False), (128, True), (256, False)])
def test_scores_are_the_oracles(O, kind, d, scaled):
    rng = np.random.default_rng(d)
    scale = O.oracle_attention_scale_q32(d) if scaled else 0
    q, k = rows(rng, (200, d), kind), rows(rng, (200, d), kind)
    with np.errstate(over="ignore"):
        got = ref.score((q.astype(np.int64) * k.astype(np.int64)).sum(1), scale)
    assert got.tolist() == [score(O, a, b, scale) for a, b in zip(q, k)]


def test_the_softmax_is_the_oracles(O):
    rng = np.random.default_rng(5)
    for n in (1, 2, 3, 64, 723, 724, 725, 1500):
        for spread in (0, 3, 3000, 400000, 40000000):
            s = rng.integers(-spread, spread + 1, n).astype(np.int32)
            assert np.array_equal(ref.weights(s.astype(np.int64)), softmax(O, s)), (n, spread)
    low = (-2**31 + rng.integers(0, 1 << 19, 300)).astype(np.int32)
    assert np.array_equal(ref.weights(low.astype(np.int64)), softmax(O, low))
    ends = np.array([2**31 - 1, -2**31, 2**31 - 1, 2**31 - 70000, 0], np.int32)
    assert np.array_equal(ref.weights(ends.astype(np.int64)), softmax(O, ends))


@pytest.mark.parametrize("kind", ["model", "wide", "full"])
@pytest.mark.parametrize("n,d,scaled", [(1, 64, True), (40, 128, True), (30, 32, False), (900, 8, True)])
def test_a_row_is_the_oracles(O, kind, n, d, scaled):
    rng = np.random.default_rng(n + d)
    scale = O.oracle_attention_scale_q32(d) if scaled else 0
    q, k, v = rows(rng, d, kind), rows(rng, (n, d), kind), rows(rng, (n, d), kind)
    with np.errstate(over="ignore"):
        assert np.array_equal(ref.attend(q, k, v, scale), attend(O, q, k, v, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,d,scaled", [(4, 2, 128, True), (2, 1, 64, False), (2, 1, 36, True),
                                                     (2, 1, 256, False)])
def test_the_kernels_rows_are_the_oracles(O, heads, kv_heads, d, scaled):
    """A packed prompt's rows, and the same tokens decoded one by one over pages."""
    import torch
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib, serving
    assert _lib.lib().q8gpu_init() == 0
    rng = np.random.default_rng(d)
    n, page, scale = 37, 16, O.oracle_attention_scale_q32(d) if scaled else 0
    q, k, v = rows(rng, (n, heads * d), "model"), rows(rng, (n, kv_heads * d), "wide"), rows(rng, (n, kv_heads * d), "wide")
    want = np.zeros_like(q)
    for i in range(n):
        for h in range(heads):
            c, g = slice(h * d, (h + 1) * d), slice(h * kv_heads // heads * d, (h * kv_heads // heads + 1) * d)
            want[i, c] = attend(O, q[i, c], k[:i + 1, g], v[:i + 1, g], scale)
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    got = serving.prompt_attention(dq, dk, dv, ints([0, n]), n, heads=heads, kv_heads=kv_heads, scale_q32=scale)
    assert np.array_equal(got.cpu().numpy(), want)
    pools = [torch.zeros((4, page, kv_heads * d), dtype=torch.int32, device="cuda") for _ in range(2)]
    table, free = ints([[-1, -1, -1]]), ints([2, 0, 3])
    for i in range(n):
        held = ints([i])
        plan = serving.page_plan(held, ints([1]), table, free[-(-i // page):].contiguous(), page, 1, parents=ints([-1]))
        serving.page_append(dk[i:i + 1], dv[i:i + 1], plan.slots, *pools)
        got = serving.tree_attention(dq[i:i + 1], *pools, plan.table, held, plan.offsets, plan.masks, 1, n, heads=heads,
                                     kv_heads=kv_heads, scale_q32=scale)
        assert np.array_equal(got[0].cpu().numpy(), want[i]), i
