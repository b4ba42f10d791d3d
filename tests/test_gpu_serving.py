"""The serving operators on the GPU against their plain 64-bit restatements
(tests/serving_reference.py): every output equal, at the sizes, layouts and
masks where they could go wrong."""
import numpy as np
import pytest

import serving_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib, serving
    assert _lib.lib().q8gpu_init() == 0, "no usable CUDA device"
    return serving


def cuda(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def values(rng, shape, kind):
    """Q16.16 values: 'model' (a few units), 'wide' (past 24 bits), 'full' (any
    int32, the extremes among them), 'zero' or 'equal' (every row the same)."""
    if kind == "zero":
        return np.zeros(shape, np.int32)
    if kind == "equal":
        return np.broadcast_to(rng.integers(-90000, 90000, shape[-1]), shape).astype(np.int32)
    if kind == "full":
        x = rng.integers(-2**31, 2**31, shape)
        return np.where(rng.random(shape) < 0.1, np.where(rng.random(shape) < 0.5, -2**31, 2**31 - 1), x).astype(np.int32)
    x = rng.normal(size=shape) * 1.2
    if kind == "wide":
        x = np.where(rng.random(shape) < 0.02, x * 300, x)
    return (x * 65536).astype(np.int32)


def scale_of(d):
    from iris_b200.shapes import attention_scale_q32
    return attention_scale_q32(d)


# ---- packed prompts -------------------------------------------------------------

PROMPTS = [
    # lengths, heads, kv_heads, head_dim, scaled, window, kind
    ([1], 4, 1, 64, False, 0, "model"),
    ([0, 1, 0, 2, 0], 4, 2, 32, True, 0, "model"),
    ([5, 64, 63, 65, 1], 8, 2, 128, True, 0, "model"),
    ([130], 4, 1, 128, True, 0, "wide"),
    ([129, 3], 4, 2, 128, True, 0, "full"),
    ([70, 129], 2, 1, 256, False, 0, "model"),
    ([70, 40], 2, 1, 256, False, 0, "full"),
    ([150, 40], 4, 1, 64, False, 17, "model"),
    ([200], 2, 2, 256, False, 96, "wide"),
    ([140, 9], 3, 1, 64, True, 0, "model"),     # a group of three
    ([90], 12, 1, 32, True, 0, "wide"),         # a group of twelve
    ([50, 20], 4, 2, 80, True, 0, "model"),     # widths between the powers of two
    ([50, 20], 4, 2, 96, True, 0, "full"),
    ([33], 2, 1, 4, True, 0, "model"),
    ([40], 2, 1, 36, False, 8, "full"),
    ([300], 4, 1, 128, True, 0, "zero"),        # all scores equal
    ([1100], 1, 1, 64, True, 0, "equal"),
    ([0, 700, 30], 2, 1, 128, True, 1, "model"),  # a window of one: every row sees itself only
    # heads of 128 values in requests of 256 rows or more
    ([257, 3, 130], 4, 1, 128, True, 0, "model"),
    ([300, 31], 2, 2, 128, False, 0, "model"),
    ([290], 8, 1, 128, True, 100, "model"),
    ([400, 17, 0, 64], 3, 1, 128, True, 33, "model"),
    ([270], 2, 1, 128, True, 0, "wide"),
    ([270, 5], 2, 1, 128, False, 0, "full"),
    ([900], 1, 1, 128, True, 0, "equal"),
    ([300, 33, 1], 2, 1, 256, False, 0, "model"),
    ([280, 100], 3, 1, 256, False, 60, "model"),
    ([260], 2, 2, 256, False, 0, "wide"),
    ([258], 2, 1, 256, True, 0, "full"),
    ([310, 7], 4, 1, 64, False, 0, "model"),
    ([256, 31], 4, 2, 96, True, 70, "model"),
    ([300], 2, 1, 160, True, 0, "model"),
    ([270], 8, 1, 32, True, 0, "model"),
]


@pytest.mark.parametrize("lengths,heads,kv_heads,d,scaled,window,kind", PROMPTS)
def test_prompt_attention_equals_the_definition(S, lengths, heads, kv_heads, d, scaled, window, kind):
    rng = np.random.default_rng(sum(lengths) + d)
    n = sum(lengths)
    q = values(rng, (n, heads * d), kind)
    k = values(rng, (n, kv_heads * d), kind)
    v = values(rng, (n, kv_heads * d), "full" if kind == "full" else "wide")
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    scale = scale_of(d) if scaled else 0
    got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), max(lengths), heads=heads, kv_heads=kv_heads,
                             scale_q32=scale, window=window).cpu().numpy()
    assert np.array_equal(got, ref.prompts(q, k, v, offsets, heads, kv_heads, scale, window))


@pytest.mark.parametrize("lengths,heads,kv_heads,d,scaled,window,kind", [c for c in PROMPTS if sum(c[0]) >= 128])
def test_prompt_attention_with_room_for_longer_requests(S, lengths, heads, kv_heads, d, scaled, window, kind):
    """`longest` is a bound: with a loose one other kernels are chosen, for the same result."""
    rng = np.random.default_rng(sum(lengths) + d + 1)
    n = sum(lengths)
    q = values(rng, (n, heads * d), kind)
    k = values(rng, (n, kv_heads * d), kind)
    v = values(rng, (n, kv_heads * d), "full" if kind == "full" else "wide" if sum(lengths) % 2 else "model")
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    scale = scale_of(d) if scaled else 0
    for longest in (1100, 20000):
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), longest, heads=heads, kv_heads=kv_heads,
                                 scale_q32=scale, window=window).cpu().numpy()
        assert np.array_equal(got, ref.prompts(q, k, v, offsets, heads, kv_heads, scale, window))


def test_weights_at_the_edge_between_two_values(S):
    """Many rows of many keys: among their weights some lie within 2^-15 of the
    edge between two values (one row of these inputs has one at 554.49996)."""
    for lengths, heads, kv_heads, d in (([5, 64, 63, 65, 1], 8, 2, 128), ([500, 501], 8, 2, 64), ([1300], 4, 1, 32)):
        rng = np.random.default_rng(sum(lengths) + d)
        n = sum(lengths)
        q, k = (values(rng, (n, w * d), "model") for w in (heads, kv_heads))
        v = values(rng, (n, kv_heads * d), "wide")
        offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        for longest in (max(lengths), 2000):
            got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), longest, heads=heads, kv_heads=kv_heads,
                                     scale_q32=scale_of(d)).cpu().numpy()
            assert np.array_equal(got, ref.prompts(q, k, v, offsets, heads, kv_heads, scale_of(d), 0))


@pytest.mark.parametrize("heads,kv_heads,d,step", [(4, 1, 128, 61), (2, 2, 64, 61), (2, 1, 36, 61), (4, 2, 128, 1),
                                                   (2, 1, 256, 61)])
def test_scores_at_the_lowest_value(S, heads, kv_heads, d, step):
    """Every score within 16.0 of the lowest one, or saturated at it: what a row
    does not see must not be told by a low score."""
    rng = np.random.default_rng(d + step)
    lengths = [300, 40]
    n = sum(lengths)
    unit = -(1 << 31) // (d << 22 >> 16)  # a key value whose score is about -2^31 against queries of 2^22
    q = np.full((n, heads * d), 1 << 22, np.int32)
    k = np.full((n, kv_heads * d), unit + step, np.int32)
    k[rng.random(n) < 0.3] += 9 if step > 1 else -3  # with a step of 1 some fall below the lowest score
    v = values(rng, (n, kv_heads * d), "model")
    offsets = np.array([0, 300, 340], np.int32)
    for window in (0, 50):
        got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(offsets), 300, heads=heads, kv_heads=kv_heads,
                                 window=window).cpu().numpy()
        assert np.array_equal(got, ref.prompts(q, k, v, offsets, heads, kv_heads, 0, window))
    for held, nodes in (([150, 0], [9, 5]), ([600, 0], [20, 13])):
        x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model", holes=[(0, 3, -1)])
        x["q"][:] = 1 << 22
        x["k_pages"][:] = unit + step
        x["k_pages"][::3] += 9 if step > 1 else -3
        x["masks"][sum(nodes) - 2] = 0
        check_tree(S, x, heads, kv_heads, 0, 0, nodes)


def test_prompt_attention_over_parts_of_fused_rows_and_a_strided_output(S):
    import torch
    rng = np.random.default_rng(3)
    heads, kv_heads, d, lengths = 4, 2, 128, [37, 100]
    n, qd, kd = sum(lengths), 512, 256
    qkv = values(rng, (n, qd + 2 * kd + 4), "model")  # four values of padding a row
    x = cuda(qkv)
    offsets = np.array([0, 37, 137], np.int32)
    out = torch.full((n, 2 * qd), 7, dtype=torch.int32, device="cuda")
    S.prompt_attention(x[:, :qd], x[:, qd:qd + kd], x[:, qd + kd:qd + 2 * kd], cuda(offsets), 100, heads=heads,
                       kv_heads=kv_heads, scale_q32=scale_of(d), out=out[:, qd:])
    want = ref.prompts(qkv[:, :qd], qkv[:, qd:qd + kd], qkv[:, qd + kd:qd + 2 * kd], offsets, heads, kv_heads,
                       scale_of(d), 0)
    assert np.array_equal(out[:, qd:].cpu().numpy(), want)
    assert (out[:, :qd] == 7).all()


def test_a_long_prompt_row_equals_its_own_attention(S):
    """Rows of a prompt past several key tiles, checked one by one (the whole prompt would take minutes on the host)."""
    rng = np.random.default_rng(8)
    heads, kv_heads, d, n = 4, 1, 128, 2500
    q, k, v = (values(rng, (n, w), "model") for w in (heads * d, d, d))
    k[1700:1710] = k[40]  # ties far apart: the first maximum counts
    q[2400:] = np.tile(k[40] * 2, 4)
    got = S.prompt_attention(cuda(q), cuda(k), cuda(v), cuda(np.array([0, n], np.int32)), n, heads=heads,
                             kv_heads=kv_heads, scale_q32=scale_of(d)).cpu().numpy()
    for i in [0, 63, 64, 127, 128, 1023, 1024, 1709, 2400, 2499]:
        for h in range(heads):
            c = slice(h * d, (h + 1) * d)
            assert np.array_equal(got[i, c], ref.attend(q[i, c], k[:i + 1], v[:i + 1], scale_of(d))), (i, h)


# ---- drafted trees over the paged cache ---------------------------------------------

def tree_inputs(rng, held, nodes, heads, kv_heads, d, page, kind, spare=2, holes=()):
    pages = [-(-(h + n) // page) for h, n in zip(held, nodes)]
    pool = sum(pages) + spare
    order = rng.permutation(pool).astype(np.int32)
    width = max(pages + [1])
    table = np.full((len(held), width), -1, np.int32)
    at = 0
    for r, p in enumerate(pages):
        table[r, :p] = order[at:at + p]
        at += p
    for r, c, what in holes:
        table[r, c] = what
    parents, masks, positions = [], [], []
    for h, n in zip(held, nodes):
        own = []
        for i in range(n):
            up = -1 if i == 0 else (i - 1 if rng.random() < 0.5 else int(rng.integers(0, i)))
            parents.append(up)
            own.append((own[up] if up >= 0 else 0) | 1 << i)
            positions.append(h + bin(own[-1]).count("1") - 1)
        masks += own
    n = sum(nodes)
    return dict(q=values(rng, (n, heads * d), kind), k_pages=values(rng, (pool, page, kv_heads * d), kind),
                v_pages=values(rng, (pool, page, kv_heads * d), "full" if kind == "full" else "wide"), table=table,
                held=np.array(held, np.int32), offsets=np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32),
                masks=np.array([m - (1 << 64) if m >> 63 else m for m in masks], np.int64),
                positions=np.array(positions, np.int32), parents=np.array(parents, np.int32))


def check_tree(S, x, heads, kv_heads, scale, window, nodes, longest=None):
    longest = longest or int((x["held"] + np.diff(x["offsets"])).max())
    got = S.tree_attention(*(cuda(x[n]) for n in ("q", "k_pages", "v_pages", "table", "held", "offsets", "masks")),
                           max(nodes), longest, heads=heads, kv_heads=kv_heads, scale_q32=scale, window=window,
                           positions=cuda(x["positions"]) if window else None).cpu().numpy()
    masks = [int(m) & (1 << 64) - 1 for m in x["masks"]]
    want = ref.trees(x["q"], x["k_pages"], x["v_pages"], x["table"], x["held"], x["offsets"], masks, x["positions"],
                     heads, kv_heads, scale, window)
    assert np.array_equal(got, want)
    return got


TREES = [
    # held, nodes, heads, kv_heads, head_dim, scaled, window, page, kind
    ([0], [1], 4, 1, 64, False, 0, 16, "model"),
    ([1], [1], 8, 2, 128, True, 0, 16, "model"),
    ([777], [1], 8, 2, 128, True, 0, 16, "wide"),
    ([100, 0, 33, 16], [13, 7, 0, 64], 8, 2, 128, True, 0, 16, "model"),
    ([257, 31], [24, 9], 8, 1, 128, True, 0, 16, "full"),
    ([90, 300], [5, 64], 2, 1, 256, False, 0, 16, "model"),
    ([200, 7, 0], [12, 20, 3], 4, 1, 64, False, 16, 16, "model"),
    ([130], [64], 2, 1, 256, False, 96, 16, "full"),
    ([61, 5], [6, 11], 4, 2, 32, True, 0, 5, "wide"),     # pages of an odd size
    ([40, 3], [3, 1], 4, 2, 32, True, 0, 1, "model"),     # pages of one token
    ([70, 64], [33, 2], 3, 1, 128, True, 0, 64, "model"),
    ([70, 9], [5, 2], 16, 1, 64, True, 0, 128, "wide"),
    ([45], [6], 4, 2, 80, True, 0, 16, "model"),
    ([45], [6], 4, 2, 36, False, 0, 16, "full"),
    ([700], [5], 4, 1, 128, True, 0, 16, "zero"),         # equal scores
    ([1500], [2], 2, 1, 64, True, 0, 16, "equal"),
    # 24 rows of a K/V head or more, heads of 128 values, 512 keys or more
    ([600, 0, 33, 515], [13, 7, 0, 24], 8, 2, 128, True, 0, 16, "model"),
    ([1030, 2], [64, 1], 2, 2, 128, True, 0, 16, "model"),
    ([520], [64], 8, 1, 128, False, 0, 16, "model"),     # 512 rows
    ([500, 700], [30, 12], 3, 1, 128, True, 100, 5, "model"),
    ([530, 64], [9, 30], 4, 1, 128, True, 0, 16, "wide"),
    ([540], [8], 4, 1, 128, False, 0, 16, "full"),
    ([900, 100], [6, 8], 4, 1, 128, True, 0, 64, "equal"),
    ([700, 20], [12, 30], 4, 2, 64, False, 200, 16, "model"),
    ([600], [10], 4, 1, 96, True, 0, 16, "model"),
    ([610, 5], [13, 8], 4, 1, 32, True, 0, 16, "wide"),
]


@pytest.mark.parametrize("held,nodes,heads,kv_heads,d,scaled,window,page,kind", TREES)
def test_tree_attention_equals_the_definition(S, held, nodes, heads, kv_heads, d, scaled, window, page, kind):
    rng = np.random.default_rng(sum(held) + d + page)
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, page, kind)
    check_tree(S, x, heads, kv_heads, scale_of(d) if scaled else 0, window, nodes)


@pytest.mark.parametrize("held,nodes,heads,kv_heads,d,scaled,window,page,kind", TREES)
def test_tree_attention_with_room_for_longer_requests(S, held, nodes, heads, kv_heads, d, scaled, window, page, kind):
    """`longest` and `nodes` are bounds: with loose ones other kernels are chosen, for the same result."""
    rng = np.random.default_rng(sum(held) + d + page + 1)
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, page, kind)
    wide = np.full((len(held), (1 << 18) // page + 1), -1, np.int32)
    wide[:, :x["table"].shape[1]] = x["table"]
    x["table"] = wide
    for most, longest in ((max(nodes), 3000), (max(nodes), (1 << 18) // (len(held) * kv_heads)), (64, 1500)):
        check_tree(S, x, heads, kv_heads, scale_of(d) if scaled else 0, window, [most],
                   max(longest, int((x["held"] + np.diff(x["offsets"])).max())))


@pytest.mark.parametrize("d", [36, 128])
def test_masks_that_leave_rows_empty_and_tables_with_holes(S, d):
    rng = np.random.default_rng(d)
    held, nodes = [0, 50, 0], [4, 8, 0]
    x = tree_inputs(rng, held, nodes, 4, 2, d, 16, "model", holes=[(1, 0, -1), (1, 2, 10**6)])
    x["masks"][1] = 0         # no cached tokens and no nodes: zeros
    x["masks"][2] = 1 << 1    # another node, not itself
    x["masks"][5] = 0         # cached tokens only
    x["masks"][6] = -1        # bits past the request's nodes name nothing
    got = check_tree(S, x, 4, 2, scale_of(d), 0, nodes)
    assert not got[1].any() and got[0].any()
    x["table"][1, :] = -1     # nothing of the request is in the pool
    got = check_tree(S, x, 4, 2, scale_of(d), 0, nodes)
    assert not got[4:].any()
    held, nodes = [0, 700, 40], [14, 12, 3]
    x = tree_inputs(rng, held, nodes, 4, 2, d, 16, "model", holes=[(1, 0, -1), (1, 30, 10**6), (1, 44, -7)])
    x["masks"][1], x["masks"][2], x["masks"][20], x["masks"][21] = 0, 1 << 1, 0, -1
    got = check_tree(S, x, 4, 2, scale_of(d), 0, nodes)
    assert not got[1].any()


@pytest.mark.parametrize("requests,nodes,most,heads,kv_heads,d,window", [
    (24, 1, 90, 8, 8, 64, 0), (9, 1, 300, 4, 4, 128, 0), (5, 2, 700, 16, 4, 128, 40), (3, 4, 500, 8, 1, 32, 0),
    (2, 1, 1500, 4, 1, 256, 0), (40, 3, 50, 4, 2, 64, 0), (1, 1, 2600, 2, 1, 128, 0)])
def test_tree_attention_of_few_rows(S, requests, nodes, most, heads, kv_heads, d, window):
    """Plain decoding and small drafts of one to many requests."""
    rng = np.random.default_rng(requests * 7 + d)
    held = [most] + [int(rng.integers(0, most + 1)) for _ in range(requests - 1)]
    sizes = [nodes] + [int(rng.integers(0, nodes + 1)) for _ in range(requests - 1)]
    for kind in ("model", "wide" if requests < 10 else "full"):
        x = tree_inputs(rng, held, sizes, heads, kv_heads, d, 16, kind, holes=[(0, 1, -1)] if most > 40 else ())
        check_tree(S, x, heads, kv_heads, scale_of(d), window, sizes)


def test_tree_attention_of_a_long_context(S):
    rng = np.random.default_rng(21)
    held, nodes, heads, kv_heads, d = [20000, 9000], [3, 2], 2, 1, 128
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model")
    check_tree(S, x, heads, kv_heads, scale_of(d), 0, nodes)


def test_tree_attention_of_wide_trees_over_a_long_context(S):
    rng = np.random.default_rng(22)
    held, nodes, heads, kv_heads, d = [9000, 4100], [7, 3], 4, 1, 128
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model")
    check_tree(S, x, heads, kv_heads, scale_of(d), 0, nodes)
    check_tree(S, x, heads, kv_heads, scale_of(d), 6000, nodes)


def test_drafted_rows_equal_one_by_one_decoding(S):
    """Every node's row equals the row of its path decoded as plain single tokens."""
    rng = np.random.default_rng(4)
    heads, kv_heads, d, held, n = 8, 2, 128, 60, 10
    x = tree_inputs(rng, [held], [n], heads, kv_heads, d, 16, "model")
    got = check_tree(S, x, heads, kv_heads, scale_of(d), 0, [n])
    flat_k, flat_v = (x[c].reshape(-1, kv_heads * d) for c in ("k_pages", "v_pages"))
    rows = [int(x["table"][0, t // 16]) * 16 + t % 16 for t in range(held + n)]
    for i in range(n):
        path = [j for j in range(n) if int(x["masks"][i]) >> j & 1]
        order = [rows[t] for t in range(held)] + [rows[held + j] for j in path]
        m = len(order)
        pages = -(-m // 16)
        k1, v1 = (np.zeros((pages * 16, kv_heads * d), np.int32) for _ in range(2))
        k1[:m], v1[:m] = flat_k[order], flat_v[order]
        one = S.tree_attention(cuda(x["q"][i:i + 1]), cuda(k1.reshape(pages, 16, -1)), cuda(v1.reshape(pages, 16, -1)),
                               cuda(np.arange(pages, dtype=np.int32)[None]), cuda(np.array([m - 1], np.int32)),
                               cuda(np.array([0, 1], np.int32)), cuda(np.array([1], np.int64)), 1, m, heads=heads,
                               kv_heads=kv_heads, scale_q32=scale_of(d)).cpu().numpy()
        assert np.array_equal(one[0], got[i])


# ---- plan, append, accept -----------------------------------------------------------

PLANS = [
    # requests, most held, most fresh, page, with parents
    (1, 0, 1, 16, False), (1, 40, 1, 16, True), (7, 100, 30, 16, True), (64, 0, 200, 16, False),
    (300, 50, 64, 5, True), (1500, 3000, 12, 64, False), (9000, 10, 3, 1, False), (16384, 5, 2, 16, False),
]


@pytest.mark.parametrize("requests,held,fresh,page,tree", PLANS)
def test_page_plan_equals_the_definition(S, requests, held, fresh, page, tree):
    rng = np.random.default_rng(requests)
    h = rng.integers(0, held + 1, requests).astype(np.int32)
    f = np.where(rng.random(requests) < 0.2, 0, rng.integers(1, fresh + 1, requests)).astype(np.int32)
    before, after = -(-h // page), -(-(h + f) // page)
    width = int(max(after.max(), 1))
    order = rng.permutation(int(after.sum()) + 5).astype(np.int32)
    table = np.full((requests, width), -1, np.int32)
    at = 0
    for r in range(requests):
        table[r, :before[r]] = order[at:at + before[r]]
        at += before[r]
    free = order[at:]
    total = int(f.sum())
    parents = None
    if tree:
        parents = np.concatenate([[int(rng.integers(-1, i)) if i else -1 for i in range(n)] for n in f] or [[]]).astype(np.int32)
    tokens = total + 3
    want = ref.plan(h, f, table, free, page, tokens, parents)
    got = S.page_plan(cuda(h), cuda(f), cuda(table), cuda(free), page, tokens,
                      parents=cuda(np.concatenate([parents, [0, 0, 0]]).astype(np.int32)) if tree else None)
    for a, b in zip((got.offsets, got.slots, got.positions, got.table), want):
        assert np.array_equal(a.cpu().numpy(), b)
    assert got.counts.tolist() == [total, want[4], 0, 0] and got.faults() == 0
    if tree:
        assert np.array_equal(got.masks.cpu().numpy(), want[5])


def test_page_plan_reports_what_does_not_fit(S):
    from iris_b200 import _lib
    held, fresh = np.array([3, 0, 20], np.int32), np.array([30, 9, 5], np.int32)
    table = np.full((3, 3), -1, np.int32)
    table[0, 0], table[2, :2] = 9, (4, 5)
    # a pool of two free pages where four are needed
    want = ref.plan(held, fresh, table, np.array([7, 8]), 16, 44)
    got = S.page_plan(cuda(held), cuda(fresh), cuda(table), cuda(np.array([7, 8], np.int32)), 16, 44)
    assert got.faults() == _lib.PLAN_POOL and got.counts.tolist()[:3] == [44, 3, 0]
    for a, b in zip((got.offsets, got.slots, got.positions, got.table), want):
        assert np.array_equal(a.cpu().numpy(), b)
    assert (got.slots.cpu().numpy()[30:39] == -1).all()
    # a table too narrow, and fewer rows than tokens
    narrow = table[:, :2].copy()
    want = ref.plan(held, fresh, narrow, np.arange(20, 30), 16, 40)
    got = S.page_plan(cuda(held), cuda(fresh), cuda(narrow), cuda(np.arange(20, 30, dtype=np.int32)), 16, 40)
    assert got.faults() == _lib.PLAN_WIDTH | _lib.PLAN_TOKENS and got.counts.tolist()[:3] == [44, 3, 4]
    for a, b in zip((got.offsets, got.slots, got.positions, got.table), want):
        assert np.array_equal(a.cpu().numpy(), b)
    # negative lengths count as none
    got = S.page_plan(cuda(np.array([-5, 2], np.int32)), cuda(np.array([2, -1], np.int32)),
                      cuda(np.array([[-1], [3]], np.int32)), cuda(np.array([6], np.int32)), 16, 2)
    assert got.faults() == _lib.PLAN_LENGTH and got.slots.tolist() == [96, 97]


def test_page_plan_with_parents_that_are_no_tree(S):
    held, fresh = np.array([4], np.int32), np.array([70], np.int32)
    parents = np.array([-1, 0, 2, 2, 7, 1, -2, -1] + [0] * 62, np.int32)  # 2 and 4 hang on no earlier node, 6 on nothing
    table = np.arange(5, dtype=np.int32)[None]
    got = S.page_plan(cuda(held), cuda(fresh), cuda(table), cuda(np.zeros(0, np.int32)), 16, 70, parents=cuda(parents))
    table[0, 1:] = -1
    m = got.masks.tolist()
    assert m[:8] == [1, 3, 0, 0, 0, 1 | 2 | 32, 0, 128]
    assert m[8] == 1 | 1 << 8 and m[63] == 1 | -(1 << 63) and m[64:] == [0] * 6
    assert got.positions.tolist()[:8] == [4, 5, 6, 7, 8, 6, 10, 4] and got.positions.tolist()[69] == 73


@pytest.mark.parametrize("tokens,kv_dim,stride", [(1, 4, 4), (61, 1024, 3072), (500, 36, 40), (3001, 64, 64)])
def test_page_append_copies_rows_to_their_slots(S, tokens, kv_dim, stride):
    import torch
    rng = np.random.default_rng(tokens)
    k, v = (rng.integers(-2**31, 2**31, (tokens, stride)).astype(np.int32) for _ in range(2))
    pages, page = tokens // 16 + 4, 16
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[::7] = -1
    slots[3::11] = pages * page  # past the pool
    pools = [np.full((pages, page, kv_dim), 5, np.int32) for _ in range(2)]
    got = [cuda(p) for p in pools]
    S.page_append(cuda(k)[:, :kv_dim], cuda(v)[:, :kv_dim], cuda(slots), *got)
    ok = (slots >= 0) & (slots < pages * page)
    for p, x in zip(pools, (k, v)):
        p.reshape(-1, kv_dim)[slots[ok]] = x[ok, :kv_dim]
    assert np.array_equal(got[0].cpu().numpy(), pools[0]) and np.array_equal(got[1].cpu().numpy(), pools[1])
    S.page_append(torch.empty((0, kv_dim), dtype=torch.int32, device="cuda"),
                  torch.empty((0, kv_dim), dtype=torch.int32, device="cuda"), cuda(np.zeros(0, np.int64)), *got)
    assert np.array_equal(got[0].cpu().numpy(), pools[0])


@pytest.mark.parametrize("requests,nodes,layers,kv_dim,page", [(1, 1, 1, 4, 16), (5, 13, 1, 64, 16), (9, 64, 3, 36, 5),
                                                              (3, 64, 2, 1024, 16)])
def test_tree_accept_equals_the_walk(S, requests, nodes, layers, kv_dim, page):
    rng = np.random.default_rng(nodes + layers)
    sizes = [nodes] + [int(rng.integers(0, nodes + 1)) for _ in range(requests - 1)]
    held = rng.integers(0, 40, requests)
    x = tree_inputs(rng, list(held), sizes, 1, 1, kv_dim, page, "model")
    offsets = x["offsets"]
    tokens = rng.integers(0, 4, offsets[-1]).astype(np.int32)  # many siblings of one token
    picks = rng.integers(0, 4, offsets[-1]).astype(np.int32)
    parents = x["parents"].copy()
    parents[parents.size // 2:][::5] = 63  # no earlier node: never accepted
    parents[offsets[:-1][np.diff(offsets) > 0]] = -1
    pools = [rng.integers(-9, 9, (layers, *x["k_pages"].shape)).astype(np.int32) for _ in range(2)]
    got_pools = [cuda(p) for p in pools]
    args = [cuda(a) for a in (tokens, parents, picks, offsets, x["held"], x["table"])]
    got = S.tree_accept(*args, 64, k_pages=got_pools[0], v_pages=got_pools[1])
    alone = S.tree_accept(*args, 64)
    for r in range(requests):
        a, b = offsets[r], offsets[r + 1]
        path = ref.walk(parents[a:b], tokens[a:b], picks[a:b])
        want = path + [-1] * (64 - len(path))
        for g in (got, alone):
            assert g.path[r].tolist() == want
            assert int(g.accepted[r]) == len(path) and int(g.held[r]) == held[r] + len(path)
            assert int(g.next[r]) == (picks[a + path[-1]] if path else -1)
        for p in pools:
            flat = p.reshape(layers, -1, kv_dim)
            at = [[int(x["table"][r, (held[r] + t) // page]) * page + (held[r] + t) % page for t in n]
                  for n in (path, range(len(path)))]
            flat[:, at[1]] = flat[:, at[0]].copy()
    for g, p in zip(got_pools, pools):
        assert np.array_equal(g.cpu().numpy(), p)


# ---- streams, graphs -----------------------------------------------------------------

def test_another_stream_and_a_captured_step(S):
    """Plan, append, tree attention and acceptance on a stream of their own,
    then replayed from a graph on new inputs."""
    import torch
    rng = np.random.default_rng(11)
    heads, kv_heads, d, held, nodes = 8, 2, 128, [100, 37], [13, 5]
    x = tree_inputs(rng, held, nodes, heads, kv_heads, d, 16, "model")
    full = x["table"].copy()
    before, after = [-(-h // 16) for h in held], [-(-(h + n) // 16) for h, n in zip(held, nodes)]
    free = np.concatenate([full[r, b:a] for r, (b, a) in enumerate(zip(before, after))])
    for r, b in enumerate(before):
        x["table"][r, b:] = -1
    rows = sum(nodes)
    dev = {n: cuda(a) for n, a in x.items()}
    dev["free"], dev["fresh"] = cuda(free), cuda(np.array(nodes, np.int32))
    dev["k"], dev["v"] = (cuda(values(rng, (rows, kv_heads * d), "model")) for _ in range(2))
    dev["tokens"], dev["picks"] = (cuda(rng.integers(0, 3, rows).astype(np.int32)) for _ in range(2))

    def step():
        p = S.page_plan(dev["held"], dev["fresh"], dev["table"], dev["free"], 16, rows, parents=dev["parents"])
        S.page_append(dev["k"], dev["v"], p.slots, dev["k_pages"], dev["v_pages"])
        o = S.tree_attention(dev["q"], dev["k_pages"], dev["v_pages"], p.table, dev["held"], p.offsets, p.masks, 13,
                             113, heads=heads, kv_heads=kv_heads, scale_q32=scale_of(d))
        return p, o, S.tree_accept(dev["tokens"], dev["parents"], dev["picks"], p.offsets, dev["held"], p.table, 16)

    def check(plan, out, done):
        torch.cuda.synchronize()
        assert np.array_equal(plan.table.cpu().numpy(), full) and plan.faults() == 0
        assert np.array_equal(plan.masks.cpu().numpy(), x["masks"])
        got = {n: dev[n].cpu().numpy() for n in ("q", "k_pages", "v_pages", "tokens", "picks")}
        want = ref.trees(got["q"], got["k_pages"], got["v_pages"], full, x["held"], x["offsets"],
                         [int(m) for m in x["masks"]], x["positions"], heads, kv_heads, scale_of(d), 0)
        assert np.array_equal(out.cpu().numpy(), want)
        for r in range(2):
            a, b = x["offsets"][r], x["offsets"][r + 1]
            path = ref.walk(x["parents"][a:b], got["tokens"][a:b], got["picks"][a:b])
            assert done.path[r].tolist() == path + [-1] * (16 - len(path))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    check(*first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        again = step()
    dev["q"].copy_(cuda(values(rng, x["q"].shape, "model")))
    dev["k"].copy_(cuda(values(rng, tuple(dev["k"].shape), "wide")))
    dev["tokens"].copy_(cuda(rng.integers(0, 3, rows).astype(np.int32)))
    g.replay()
    check(*again)


def test_a_pool_of_more_than_32_bits_of_values(S):
    """Pages past 2^32 values into the pools: appended, attended over and moved as in a small pool."""
    import torch
    rng = np.random.default_rng(31)
    heads, kv_heads, d, page, pages = 16, 8, 128, 16, 270000  # 17.7 GB a pool
    width = kv_heads * d
    assert (pages - 1) * page * width > 1 << 32
    free, _ = torch.cuda.mem_get_info()
    if free < 45 << 30:
        pytest.skip("needs 45 GB")
    big_k, big_v = (torch.empty((pages, page, width), dtype=torch.int32, device="cuda") for _ in range(2))
    for held, nodes in ((700, 1), (300, 6), (700, 12), (700, 40), (4200, 3)):
        x = tree_inputs(rng, [held], [nodes], heads, kv_heads, d, page, "model", spare=0)
        n = held + nodes
        used = x["table"].shape[1]
        ids = (pages - used + rng.permutation(used)).astype(np.int32)  # the pool's last pages
        ids[0] = 3
        rows = [int(x["table"][0, t // page]) * page + t % page for t in range(n)]
        slots = np.array([int(ids[t // page]) * page + t % page for t in range(n)], np.int64)
        k, v = (x[name].reshape(-1, width)[rows] for name in ("k_pages", "v_pages"))
        S.page_append(cuda(k), cuda(v), cuda(slots), big_k, big_v)
        args = [cuda(x[name]) for name in ("held", "offsets", "masks")]
        small = S.tree_attention(cuda(x["q"]), cuda(x["k_pages"]), cuda(x["v_pages"]), cuda(x["table"]), *args, nodes, n,
                                 heads=heads, kv_heads=kv_heads, scale_q32=scale_of(d))
        large = S.tree_attention(cuda(x["q"]), big_k, big_v, cuda(ids[None]), *args, nodes, n, heads=heads,
                                 kv_heads=kv_heads, scale_q32=scale_of(d))
        assert torch.equal(small, large)
        # every node accepted along its last path, in both pools
        tokens = np.arange(nodes, dtype=np.int32)
        picks = np.full(nodes, -5, np.int32)
        at = nodes - 1
        while x["parents"][at] >= 0:
            picks[x["parents"][at]] = at
            at = x["parents"][at]
        pools = [cuda(x["k_pages"])[None], cuda(x["v_pages"])[None]]
        for pk, pv, table in ((*pools, x["table"]), (big_k[None], big_v[None], ids[None])):
            done = S.tree_accept(cuda(tokens), cuda(x["parents"]), cuda(picks), args[1], args[0], cuda(table), nodes,
                                 k_pages=pk, v_pages=pv)
        moved = int(done.held[0])
        assert moved == held + bin(int(x["masks"][nodes - 1]) & (1 << 64) - 1).count("1")
        for small_pool, big in zip(pools, (big_k, big_v)):
            a = small_pool.view(-1, width)[torch.tensor(rows[:moved], device="cuda")]
            b = big.view(-1, width)[torch.from_numpy(slots[:moved]).cuda()]
            assert torch.equal(a, b)


def test_no_wait_gave_up(S):
    """The bounded waits of every call above held; the check reports a status, not a leftover."""
    S.stall_check()
    S.stall_check()
