"""The serving operators on the GPU at the edges of their ranges, against the
plain 64-bit restatements (tests/serving_reference.py)."""
import numpy as np
import pytest

import serving_reference as ref
from test_gpu_serving import PROMPTS, cuda, scale_of, tree_inputs, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib, serving
    assert _lib.lib().q8gpu_init() == 0, "no usable CUDA device"
    return serving


def run_tree(S, x, heads, kv_heads, scale, window, nodes, longest, out=None):
    return S.tree_attention(*(cuda(x[n]) for n in ("q", "k_pages", "v_pages", "table", "held", "offsets", "masks")),
                            nodes, longest, heads=heads, kv_heads=kv_heads, scale_q32=scale, window=window,
                            positions=cuda(x["positions"]) if window else None, out=out).cpu().numpy()


def tree_rows(x, heads, kv_heads, scale, window):
    return ref.trees(x["q"], x["k_pages"], x["v_pages"], x["table"], x["held"], x["offsets"],
                     [int(m) & (1 << 64) - 1 for m in x["masks"]], x["positions"], heads, kv_heads, scale, window)


@pytest.mark.parametrize("d", [32, 64, 128, 256, 36])
def test_a_sum_at_the_top_of_64_bits_is_the_highest_score(S, d):
    """A key whose unscaled sum is 2^63 - 1 among keys of small ones: its score is the highest there is."""
    rng = np.random.default_rng(d)
    heads, kv_heads = 2, 1
    row = np.zeros(d, np.int32)
    row[:3] = -2**31, -2**31, 2**31 - 1
    best, other = np.zeros(d, np.int32), np.zeros(d, np.int32)
    best[:3] = -2**31, -(2**31 - 1), 1
    other[2] = 1
    assert int((row.astype(object) * best.astype(object)).sum()) == 2**63 - 1
    n = 90
    q, k, v = np.tile(row, (n, heads)), np.tile(other, (n, 1)), values(rng, (n, d), "model")
    k[0] = best
    offsets = np.array([0, n], np.int32)
    got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), n, heads=heads, kv_heads=kv_heads).cpu().numpy()
    assert np.array_equal(got, ref.prompts(q, k, v, offsets, heads, kv_heads, 0, 0))
    assert np.array_equal(got[-1], np.tile(v[0], heads))
    for held, nodes in ((50, 1), (50, 9), (1500, 3), (400, 40)):  # in clusters, on mma.sync, on the tensor cores
        x = tree_inputs(rng, [held], [nodes], heads, kv_heads, d, 16, "model")
        x["q"][:] = np.tile(row, heads)
        x["k_pages"][:] = other
        x["k_pages"][x["table"][0, 1], 3] = best
        got = run_tree(S, x, heads, kv_heads, 0, 0, nodes, held + nodes)
        assert np.array_equal(got, tree_rows(x, heads, kv_heads, 0, 0)), (held, nodes)


@pytest.mark.parametrize("lengths,heads,kv_heads,d", [([5, 64, 300, 1], 8, 2, 128), ([130], 4, 1, 256), ([40, 3], 4, 2, 32),
                                                      ([50, 90], 4, 2, 36)])
def test_any_bound_on_the_prompts_gives_the_same_rows(S, lengths, heads, kv_heads, d):
    rng = np.random.default_rng(d)
    n = sum(lengths)
    q, k, v = (values(rng, (n, w * d), "model") for w in (heads, kv_heads, kv_heads))
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    for window in (0, 24):
        want = ref.prompts(q, k, v, offsets, heads, kv_heads, scale_of(d), window)
        for longest in (max(lengths), n, n + 1, 20000, 1 << 31, 0xFFFFFF72, 0xFFFFFFFF):
            got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), longest, heads=heads, kv_heads=kv_heads,
                                     scale_q32=scale_of(d), window=window).cpu().numpy()
            assert np.array_equal(got, want), (window, longest)


@pytest.mark.parametrize("lengths,heads,kv_heads,d,scaled,window,kind",
                         [c for c in PROMPTS if c[3] % 32 == 0 and sum(c[0]) < 500])
def test_prompts_behind_a_long_one(S, lengths, heads, kv_heads, d, scaled, window, kind):
    """With a request of 1,024 rows among them the others go through the tensor cores' tiles too."""
    rng = np.random.default_rng(sum(lengths) + d + 2)
    lengths = [*lengths[:1], 1024, *lengths[1:]]
    n = sum(lengths)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    scale = scale_of(d) if scaled else 0
    for values_kind in ("model", "full" if kind == "full" else "wide"):
        q, k = (values(rng, (n, w * d), kind) for w in (heads, kv_heads))
        v = values(rng, (n, kv_heads * d), values_kind)
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), 1024, heads=heads, kv_heads=kv_heads,
                                 scale_q32=scale, window=window).cpu().numpy()
        a, b = offsets[1], offsets[2]
        short = np.r_[0:a, b:n]
        at = np.concatenate([offsets[:2], offsets[3:] - 1024])
        assert np.array_equal(got[short], ref.prompts(q[short], k[short], v[short], at, heads, kv_heads, scale, window))
        for i in [0, 1, 63, 127, 128, 500, 1023]:
            lo = a + (max(0, i + 1 - window) if window else 0)
            for h in range(heads):
                c, g = slice(h * d, (h + 1) * d), slice(h * kv_heads // heads * d, (h * kv_heads // heads + 1) * d)
                assert np.array_equal(got[a + i, c], ref.attend(q[a + i, c], k[lo:a + i + 1, g], v[lo:a + i + 1, g], scale)), i


@pytest.mark.parametrize("d", [36, 64, 128])
def test_a_window_past_every_position_hides_nothing(S, d):
    rng = np.random.default_rng(d)
    heads, kv_heads = 4, 2
    for held, nodes in (([50, 3], [5, 2]), ([1500], [4]), ([400], [40])):
        x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model")
        want = tree_rows(x, heads, kv_heads, scale_of(d), 0)
        for window in ((1 << 31) - 1, 1 << 31, (1 << 32) - 600, (1 << 32) - 1):
            got = run_tree(S, x, heads, kv_heads, scale_of(d), window, max(nodes), max(held) + max(nodes))
            assert np.array_equal(got, want), (held, window)
    q, k, v = (values(rng, (150, w * d), "model") for w in (heads, kv_heads, kv_heads))
    offsets = np.array([0, 20, 150], np.int32)
    want = ref.prompts(q, k, v, offsets, heads, kv_heads, scale_of(d), 0)
    for window in (1 << 31, (1 << 32) - 1):
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), 130, heads=heads, kv_heads=kv_heads,
                                 scale_q32=scale_of(d), window=window).cpu().numpy()
        assert np.array_equal(got, want), window


@pytest.mark.parametrize("fresh,fault", [([1 << 22] * 1024, True), ([1 << 30] * 3, True), ([1 << 30, 1 << 30], True),
                                         ([0, 1 << 30] * 600, True), ([1 << 30, (1 << 30) - 1], False),
                                         ([(1 << 31) - 1], False)])
def test_page_plan_tells_when_the_fresh_tokens_pass_31_bits(S, fresh, fault):
    """A sum of 2^31 tokens or more, over one request's run or many, is a fault of lengths."""
    from iris_b200 import _lib
    n, page = len(fresh), 1 << 20
    table = np.full((n, 2048), -1, np.int32)
    plan = S.page_plan(cuda(np.zeros(n, np.int32)), cuda(np.array(fresh, np.int32)), cuda(table),
                       cuda(np.arange(8192, dtype=np.int32)), page, 8)
    assert bool(plan.faults() & _lib.PLAN_LENGTH) == fault
    assert plan.faults() & _lib.PLAN_TOKENS or fault


def test_pages_that_no_request_names_do_not_choose_the_path(S):
    """Keys past a request's end and holes in its table stand for no row: values
    past 24 bits in the pool's first page, which no table names, leave the call on
    the tensor cores (the scratch's last words tell of such values)."""
    import ctypes as C

    import torch
    from iris_b200 import _lib
    rng = np.random.default_rng(7)
    heads, kv_heads, d, held, nodes = 4, 1, 128, [500, 130], [40, 11]
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model", holes=[(0, 2, -1), (0, 5, 1 << 20)])
    x["v_pages"] = values(rng, x["k_pages"].shape, "model")
    x["table"][x["table"] == 0] = x["k_pages"].shape[0] - 1  # page 0 is nobody's
    for where, flags in (((), [0, 0]), (("k_pages",), [1, 0]), (("v_pages",), [0, 1]), (("q",), [1, 0])):
        for name in ("k_pages", "v_pages"):
            x[name][0] = 1 << 30
        y = {n: a.copy() for n, a in x.items()}
        for name in where:  # one wide value that the call does see
            y[name].reshape(-1)[0 if name == "q" else int(x["table"][0, 1]) * 16 * d] = 1 << 28
        dev = {n: cuda(a) for n, a in y.items()}
        out = torch.empty((sum(nodes), heads * d), dtype=torch.int32, device="cuda")
        a = _lib.TreeAttention(*(dev[n].data_ptr() for n in ("q", "k_pages", "v_pages", "table", "held", "offsets",
                                                             "masks")), None, out.data_ptr(), heads * d, heads * d,
                               y["k_pages"].shape[0], len(held), sum(nodes), y["table"].shape[1], 16, max(nodes),
                               max(h + n for h, n in zip(held, nodes)), heads, kv_heads, d, 0, scale_of(d))
        need = _lib.lib().iris_tree_attention_workspace(C.byref(a))
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        _lib.check(_lib.lib().iris_tree_attention(C.byref(a), work.data_ptr(), need,
                                                  torch.cuda.current_stream().cuda_stream), "iris_tree_attention")
        assert np.array_equal(out.cpu().numpy(), tree_rows(y, heads, kv_heads, scale_of(d), 0))
        assert work[need - 256:need - 248].view(torch.int32).ne(0).int().tolist() == flags, where


def test_a_single_row_of_any_stride(S):
    """One row has no distance to the next: torch's number for it may be 1, or anything."""
    import torch
    rng = np.random.default_rng(1)
    heads, kv_heads, d = 4, 2, 64

    def one(width):
        x = values(rng, (1, width), "model")
        return x, cuda(x.reshape(-1, 1)).t()  # strides (1, 1)

    (q, dq), (k, dk), (v, dv) = one(heads * d), one(kv_heads * d), one(kv_heads * d)
    out = torch.zeros(heads * d, 1, dtype=torch.int32, device="cuda").t()
    assert dq.stride() == out.stride() == (1, 1)
    offsets = np.array([0, 1], np.int32)
    S.prompt_attention(dq, dk, dv, cuda(offsets), 1, heads=heads, kv_heads=kv_heads, out=out)
    assert np.array_equal(out.cpu().numpy(), ref.prompts(q, k, v, offsets, heads, kv_heads, 0, 0))
    pools = [torch.zeros((1, 16, kv_heads * d), dtype=torch.int32, device="cuda") for _ in range(2)]
    S.page_append(dk, dv, cuda(np.array([5])), *pools)
    assert np.array_equal(pools[0][0, 5].cpu().numpy(), k[0]) and np.array_equal(pools[1][0, 5].cpu().numpy(), v[0])
    pools[0][0, 0], pools[1][0, 0] = dk[0], dv[0]
    out.zero_()
    S.tree_attention(dq, *pools, cuda(np.zeros((1, 1), np.int32)), cuda(np.zeros(1, np.int32)), cuda(offsets),
                     cuda(np.ones(1, np.int64)), 1, 1, heads=heads, kv_heads=kv_heads, out=out)
    assert np.array_equal(out.cpu().numpy(), ref.prompts(q, k, v, offsets, heads, kv_heads, 0, 0))


@pytest.mark.parametrize("d", [36, 64, 128])
def test_rows_of_no_request_are_left_alone(S, d):
    """Rows from the last request's end on (a step planned with room to spare) are not written, whichever kernel runs."""
    rng = np.random.default_rng(d)
    heads, kv_heads, spare = 4, 2, 5
    for held, nodes in (([50, 3], [5, 2]), ([1500], [4]), ([400], [40])):
        x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model")
        want = tree_rows(x, heads, kv_heads, scale_of(d), 0)
        n = sum(nodes)
        x["q"] = np.concatenate([x["q"], values(rng, (spare, heads * d), "model")])
        x["masks"] = np.concatenate([x["masks"], np.zeros(spare, np.int64)])
        out = cuda(np.full((n + spare, heads * d), 7, np.int32))
        got = run_tree(S, x, heads, kv_heads, scale_of(d), 0, max(nodes), max(held) + max(nodes), out=out)
        assert np.array_equal(got[:n], want) and (got[n:] == 7).all(), held
    for lengths in ([20, 45], [150, 0, 33], [1030]):
        n = sum(lengths)
        q, k, v = (values(rng, (n + spare, w * d), "model") for w in (heads, kv_heads, kv_heads))
        offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        out = cuda(np.full((n + spare, heads * d), 7, np.int32))
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), max(lengths), heads=heads, kv_heads=kv_heads,
                                 scale_q32=scale_of(d), out=out).cpu().numpy()
        assert np.array_equal(got[:n], ref.prompts(q[:n], k[:n], v[:n], offsets, heads, kv_heads, scale_of(d), 0))
        assert (got[n:] == 7).all(), lengths


def test_trees_with_a_bound_past_67_million_keys(S):
    """The widest table: the row kernel takes what the launches' grids cannot."""
    rng = np.random.default_rng(9)
    x = tree_inputs(rng, [20], [2], 2, 1, 64, 16, "model")
    table = np.full((1, (1 << 27) // 16 - 1), -1, np.int32)
    table[:, :x["table"].shape[1]] = x["table"]
    x["table"] = table
    for longest in (65535 * 1024, 65535 * 1024 + 1, (1 << 27) - 16):
        got = run_tree(S, x, 2, 1, scale_of(64), 0, 2, longest)
        assert np.array_equal(got, tree_rows(x, 2, 1, scale_of(64), 0)), longest


@pytest.mark.parametrize("n,heads,d,window,kind", [(16256, 1, 128, 0, "model"), (16257, 1, 64, 0, "model"),
                                                   (17000, 2, 32, 0, "wide"), (17000, 1, 32, 16700, "model"),
                                                   (33000, 1, 32, 0, "model")])
def test_prompts_at_and_past_the_longest_of_the_tensor_cores(S, n, heads, d, window, kind):
    """Rows past 16,256 keys, and past the 16,384 that one int32 accumulator holds, checked one by one."""
    rng = np.random.default_rng(n + d)
    q, k = (values(rng, (n, w * d), "model") for w in (heads, 1))
    v = values(rng, (n, d), kind)
    k[16200:16220] = k[3]              # ties far apart: the first maximum counts
    v[100:] = np.abs(v[100:]) + 5000000  # large sums of one sign
    got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(np.array([0, n], np.int32)), n, heads=heads, kv_heads=1,
                             scale_q32=scale_of(d), window=window).cpu().numpy()
    for i in [0, 5, 127, 128, 16127, n - 65, n - 2, n - 1]:
        lo = max(0, i + 1 - window) if window else 0
        for h in range(heads):
            c = slice(h * d, (h + 1) * d)
            assert np.array_equal(got[i, c], ref.attend(q[i, c], k[lo:i + 1], v[lo:i + 1], scale_of(d))), (i, h)


@pytest.mark.parametrize("d", [32, 36, 256])
def test_prompts_of_more_requests_than_are_sorted(S, d):
    rng = np.random.default_rng(d)
    lengths = rng.choice([0, 1, 2, 3, 9], 1100)
    lengths[700] = 130
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    n = int(offsets[-1])
    q, k, v = (values(rng, (n, w * d), "model") for w in (2, 1, 1))
    got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), 130, heads=2, kv_heads=1,
                             scale_q32=scale_of(d)).cpu().numpy()
    assert np.array_equal(got, ref.prompts(q, k, v, offsets, 2, 1, scale_of(d), 0))


def test_numbers_may_be_numpys(S):
    """Bounds taken from numpy's arrays, next to a scale of 2^31 (heads of four values)."""
    rng = np.random.default_rng(2)
    q, k, v = (values(rng, (9, w), "model") for w in (8, 4, 4))
    offsets = np.array([0, 4, 9], np.int32)
    want = ref.prompts(q, k, v, offsets, 2, 1, 1 << 31, 0)
    assert scale_of(4) == 1 << 31
    for number in (np.int32, np.uint32, np.int64, np.uint8):
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), number(5), heads=number(2),
                                 kv_heads=number(1), scale_q32=scale_of(4), window=number(0))
        assert np.array_equal(got.cpu().numpy(), want)
