"""The serving operators, measured: a step's bookkeeping on the GPU, K/V rows
into pages, packed prompt attention, attention of drafted trees over the paged
cache, and the acceptance of drafted tokens.

Every value is an integer of the framework's fixed-point formats: activations
and K/V are Q16.16 in int32, dot products and softmax sums Q32.32 in int64
(that is the operators' definition, so the plain forms hold them in 64 bits
too). Outputs are whole numbers and have exactly one right value.

Formulas (x >>r s: x / 2^s rounded to nearest, ties to even; sat: to int32):

  score   s_t = sat(floor(sum_d q_d k_td * scale / 2^32) >>r 16), scale =
          floor(2^32 / sqrt(d)); without a scale (gemma-dense) s_t =
          sat(sum_d q_d k_td >>r 16); the sum wraps at 64 bits
  term    e_t = the Q32.32 exponential of s_t - max s: with -delta = k ln2 + r,
          (1 - r + r^2/2 - r^3/6 + r^4/24 - r^5/120) >>r k, each power and
          quotient rounded to Q32.32; 0 from 16.0 below the maximum
  weight  w_t = (e_t * 2^32 / sum e, rounded to even) >>r 16; the first
          maximum's weight takes 65536 - sum w besides
  out_d   sat(sum_t w_t v_td >>r 16); a row that sees no key gives zeros
"""
import math
import random

import torch

own = False

PAGE = 16          # tokens a page
VOCAB = 32000
MAX_NODES = 64     # drafted tokens a request at most


# ---- cases ------------------------------------------------------------------

def listed():
    mistral = {"heads": 32, "kv_heads": 8, "dim": 128, "scaled": True, "window": 0}
    gemma = {"heads": 8, "kv_heads": 1, "dim": 256, "scaled": False, "window": 768}
    tiny = {"heads": 4, "kv_heads": 1, "dim": 64, "scaled": False, "window": 96}
    return [
        # a decode step of 32 requests with drafted trees: pure launch latency
        {"name": "plan a drafted step", "op": "plan", "requests": 32, "held": 4096, "fresh": 24, "tree": True, "mix": 1},
        # many prompts arrive at once: about a million slots
        {"name": "plan 4001 prompts", "op": "plan", "requests": 4001, "held": 0, "fresh": 512, "tree": False, "mix": 2},
        # the drafted tokens of one step of one layer
        {"name": "append 61 rows", "op": "append", "tokens": 61, "width": 1024, "mix": 3},
        # the prompts of a 4096-token claim and its neighbours, one layer
        {"name": "append 8191 rows", "op": "append", "tokens": 8191, "width": 1024, "mix": 4},
        # short prompts on the tiny gemma shape
        {"name": "prompts, tiny", "op": "prompt", "lengths": "32,1,96,7,33", "mix": 5, **tiny},
        # gemma-2b shape: 512-token prompts and longer ones past its window
        {"name": "prompts, gemma-2b", "op": "prompt", "lengths": "512,1025,0,37,640", "mix": 6, **gemma},
        # mistral-7b shape: the 4096-token claim packed with shorter prompts
        {"name": "prompts, mistral-7b", "op": "prompt", "lengths": "4096,300,1,1037,711", "mix": 7, **mistral},
        # plain decoding of one sequence: one node, a context of a few hundred
        {"name": "tree of one node", "op": "tree", "held": "777", "nodes": "1", "mix": 8, **mistral},
        # a serving batch with drafted trees of 1 to 24 nodes
        {"name": "trees of a batch", "op": "tree",
         "held": "2050,4095,17,0,1300,3333,512,2900,640,4000,96,1801,2222,3071,1,900",
         "nodes": "13,24,8,13,1,16,13,9,24,13,5,13,12,16,24,13", "mix": 9, **mistral},
        # wide trees over contexts near the model's 32768 positions
        {"name": "wide trees, long", "op": "tree", "held": "32001,20011", "nodes": "64,48", "mix": 10, **mistral},
        # one model's step: 16 requests, the cache of one layer
        {"name": "accept a batch", "op": "accept", "requests": 16, "nodes": 13, "layers": 1, "width": 1024, "held": 512, "mix": 11},
        # the accepted rows of every layer of mistral-7b
        {"name": "accept, 32 layers", "op": "accept", "requests": 48, "nodes": 61, "layers": 32, "width": 1024, "held": 96, "mix": 12},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "prompt", "prompt", "tree", "tree", "accept"])
    mix = rng.randrange(1 << 30)
    shape = rng.choice([{"heads": 32, "kv_heads": 8, "dim": 128, "scaled": True, "window": 0},
                        {"heads": 8, "kv_heads": 1, "dim": 256, "scaled": False, "window": rng.choice([0, 768])},
                        {"heads": 4, "kv_heads": 2, "dim": 32, "scaled": True, "window": 0},
                        {"heads": 4, "kv_heads": 1, "dim": 64, "scaled": False, "window": rng.choice([16, 96])}])
    if op == "plan":
        tree = rng.random() < 0.5
        return {"op": op, "requests": _log(rng, 1, 256 if tree else 4001), "held": rng.choice([0, _log(rng, 1, 8192)]),
                "fresh": _log(rng, 1, MAX_NODES if tree else 512), "tree": tree, "mix": mix}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 8191), "width": rng.choice([64, 256, 1024]), "mix": mix}
    if op == "prompt":
        left, lengths = _log(rng, 1, 6145), []
        while left > 0 and len(lengths) < 12:
            n = min(left, 4096, _log(rng, 1, 4096))
            lengths.append(n)
            left -= n
        rng.shuffle(lengths)
        return {"op": op, "lengths": ",".join(map(str, lengths)), "mix": mix, **shape}
    if op == "tree":
        requests = _log(rng, 1, 24)
        most = 32000 if requests <= 2 else 52000 // requests
        held = [rng.choice([0, _log(rng, 1, most), _log(rng, 1, most)]) for _ in range(requests)]
        nodes = [_log(rng, 1, MAX_NODES if requests <= 4 else 24) for _ in range(requests)]
        return {"op": op, "held": ",".join(map(str, held)), "nodes": ",".join(map(str, nodes)), "mix": mix, **shape}
    return {"op": op, "requests": _log(rng, 1, 48), "nodes": _log(rng, 1, 61), "layers": rng.choice([1, 2, 18, 32]),
            "width": rng.choice([64, 256, 1024]), "held": _log(rng, 1, 96), "mix": mix}


def _numbers(text):
    return [int(x) for x in str(text).split(",")]


def _plan_lengths(case):
    r = random.Random(case["mix"])
    held = [r.randint(0, case["held"]) for _ in range(case["requests"])]
    fresh = [r.randint(1, case["fresh"]) if r.random() < 0.9 else 0 for _ in range(case["requests"])]
    fresh[0] = case["fresh"]
    return held, fresh


def _parents(r, n):
    """A drafted tree: node 0 the last committed token, each other node under an earlier one (chains are common)."""
    return [-1 if i == 0 else (i - 1 if r.random() < 0.5 else r.randrange(i)) for i in range(n)]


def _accept_parents(case):
    r = random.Random(case["mix"])
    nodes = [max(1, case["nodes"] - r.randint(0, case["nodes"] // 2)) for _ in range(case["requests"])]
    nodes[0] = case["nodes"]
    return nodes, [_parents(r, n) for n in nodes]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def work(case):
    if case["op"] == "plan":
        held, fresh = _plan_lengths(case)
        tokens = sum(fresh)
        taken = sum(_pages(h + f) - _pages(h) for h, f in zip(held, fresh))
        # lengths in, offsets out, a table entry in or out a page, slot (8) and position (4) a token, parent and mask with trees
        return {"bytes": 12 * case["requests"] + 12 * taken + tokens * (12 + (12 if case["tree"] else 0)), "flops": 0}
    if case["op"] == "append":
        return {"bytes": case["tokens"] * (case["width"] * 16 + 8), "flops": 0}
    if case["op"] == "accept":
        nodes, _ = _accept_parents(case)
        # at least the root of every request; its rows stay, so the tree and the answers are what has to move
        moved = _accepted_moves(case)
        return {"bytes": sum(nodes) * 12 + case["requests"] * (4 * MAX_NODES + 16) + moved * case["layers"] * case["width"] * 16,
                "flops": 0}
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        lengths = _numbers(case["lengths"])
        w = case["window"] or max(lengths) + 1
        pairs = sum(min(i + 1, w) for n in lengths for i in range(n))
        return {"bytes": sum(lengths) * 8 * (H + K) * D, "flops": 4 * D * H * pairs}
    pairs, rows, keys = 0, 0, 0
    for h, n in zip(_numbers(case["held"]), _numbers(case["nodes"])):
        seen = min(h, case["window"] - 1) if case["window"] else h  # cached keys (a window reaches a little less far down the tree)
        rows += n
        keys += seen + n
        pairs += n * (seen + 1)
    return {"bytes": 8 * K * D * keys + 8 * H * D * rows, "flops": 4 * D * H * pairs}


def _accept_draft(case):
    """Token ids and picks by the case's own mix: each node's pick is one of its children's tokens half of the time."""
    nodes, parents = _accept_parents(case)
    r = random.Random(case["mix"] + 1)
    tokens, picks = [], []
    for n, p in zip(nodes, parents):
        t = [r.randrange(VOCAB) for _ in range(n)]
        k = [r.randrange(VOCAB) for _ in range(n)]
        for i in range(n):
            below = [j for j in range(n) if p[j] == i]
            if below and r.random() < 0.8:
                k[i] = t[r.choice(below)]
        tokens.append(t)
        picks.append(k)
    return nodes, parents, tokens, picks


def _walk(parents, tokens, picks):
    path = [0]
    while True:
        at = path[-1]
        below = [j for j in range(len(parents)) if parents[j] == at and tokens[j] == picks[at]]
        if not below:
            return path
        path.append(below[0])


def _accepted_moves(case):
    nodes, parents, tokens, picks = _accept_draft(case)
    return sum(1 for p, t, k in zip(parents, tokens, picks) for i, j in enumerate(_walk(p, t, k)) if i != j)


# ---- inputs -----------------------------------------------------------------

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(g, shape, sigma):
    """Q16.16 values of a normal distribution."""
    return (torch.randn(shape, generator=g, device="cuda") * (sigma * 65536)).round().clamp(-2**31, 2**31 - 1).to(torch.int32)


def _sigmas(case):
    """Queries and keys whose scores spread by about 2: scaled scores, or per-head normed ones."""
    return (1.5, 1.5) if case["scaled"] else (math.sqrt(2.0) / case["dim"] ** 0.25, math.sqrt(2.0) / case["dim"] ** 0.25)


def _scale(case):
    if not case["scaled"]:
        return 0
    return math.isqrt((1 << 64) // case["dim"])


def _tables(g, held, fresh, spare):
    """A pool in no order: the pages each request holds for its cached tokens and the fresh ones, the rest free."""
    total = [_pages(h + f) for h, f in zip(held, fresh)]
    pool = sum(total) + spare
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    width = max(total + [1])
    table = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
    counts = torch.tensor(total, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < counts[:, None]] = order[:sum(total)]
    return table, order[sum(total):], pool


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "plan":
        held, fresh = _plan_lengths(case)
        perm = torch.randperm(len(held), generator=g, device="cuda")
        r = random.Random(seed)
        parents = []
        for i in perm.tolist():
            parents += _parents(r, fresh[i])
        width = max(_pages(h + f) for h, f in zip(held, fresh)) or 1
        used = sum(_pages(h) for h in held)
        need = sum(_pages(h + f) - _pages(h) for h, f in zip(held, fresh))
        order = torch.randperm(used + need + 7, generator=g, device="cuda").to(torch.int32)
        s["held"], s["fresh"] = _i32(held)[perm], _i32(fresh)[perm]
        table = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(width, device="cuda")[None, :] < ((s["held"] + PAGE - 1) // PAGE)[:, None]] = order[:used]
        s["table"], s["free"] = table, order[used:]
        s["tokens"] = sum(fresh)
        s["parents"] = _i32(parents) if case["tree"] else None
    elif case["op"] == "append":
        n, width = case["tokens"], case["width"]
        s["k"], s["v"] = _values(g, (n, width), 1.5), _values(g, (n, width), 1.0)
        pages = _pages(n) + 8
        # requests of odd lengths: rows run on inside pages, the pages in no order; a few padded rows go nowhere
        slots = torch.arange(n, device="cuda") + 5
        order = torch.randperm(pages, generator=g, device="cuda")
        slots = order[slots // PAGE] * PAGE + slots % PAGE
        slots[torch.rand(n, generator=g, device="cuda") < 0.02] = -1
        s["slots"] = slots
        s["k_pages"] = torch.zeros((pages, PAGE, width), dtype=torch.int32, device="cuda")
        s["v_pages"] = torch.zeros((pages, PAGE, width), dtype=torch.int32, device="cuda")
    elif case["op"] == "prompt":
        lengths = _numbers(case["lengths"])
        n, H, K, D = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
        sq, sk = _sigmas(case)
        # the rows of a fused q|k|v product
        s["qkv"] = torch.cat([_values(g, (n, H * D), sq), _values(g, (n, K * D), sk), _values(g, (n, K * D), 1.0)], 1)
        s["offsets"] = _i32(_offsets(lengths))
        s["longest"] = max(lengths)
    elif case["op"] == "tree":
        held, nodes = _numbers(case["held"]), _numbers(case["nodes"])
        H, K, D = case["heads"], case["kv_heads"], case["dim"]
        sq, sk = _sigmas(case)
        table, _, pool = _tables(g, held, nodes, 3)
        r = random.Random(seed)
        parents = [_parents(r, n) for n in nodes]
        masks, positions = [], []
        for h, p in zip(held, parents):
            m = []
            for i, up in enumerate(p):
                m.append((m[up] if up >= 0 else 0) | 1 << i)
            masks += [x - (1 << 64) if x >> 63 else x for x in m]
            positions += [h + bin(x).count("1") - 1 for x in m]
        s["q"] = _values(g, (sum(nodes), H * D), sq)
        s["k_pages"], s["v_pages"] = _values(g, (pool, PAGE, K * D), sk), _values(g, (pool, PAGE, K * D), 1.0)
        s["table"], s["held"], s["offsets"] = table, _i32(held), _i32(_offsets(nodes))
        s["masks"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
        s["positions"] = _i32(positions)
        s["longest"] = max(h + n for h, n in zip(held, nodes))
        s["nodes"] = max(nodes)
    else:
        nodes, parents, tokens, picks = _accept_draft(case)
        r = random.Random(seed)
        rename = list(range(VOCAB))
        r.shuffle(rename)
        lengths = random.Random(case["mix"] + 2)
        held = [lengths.randint(0, case["held"]) for _ in nodes]
        table, _, pool = _tables(g, held, nodes, 3)
        s["tokens"] = _i32([rename[x] for t in tokens for x in t])
        s["picks"] = _i32([rename[x] for t in picks for x in t])
        s["parents"] = _i32([x for p in parents for x in p])
        s["held"], s["offsets"], s["table"] = _i32(held), _i32(_offsets(nodes)), table
        s["k_pages"] = _values(g, (case["layers"], pool, PAGE, case["width"]), 1.5)
        s["v_pages"] = _values(g, (case["layers"], pool, PAGE, case["width"]), 1.0)
    return s


def run(state):
    case = state["case"]
    return globals()["_" + ("own_" if own else "plain_") + case["op"]](case, state)


# ---- the framework's calls ----------------------------------------------------

def _own_plan(case, s):
    from iris_b200 import serving
    p = serving.page_plan(s["held"], s["fresh"], s["table"], s["free"], PAGE, s["tokens"], parents=s["parents"])
    return {"offsets": p.offsets, "slots": p.slots, "positions": p.positions, "table": p.table, "counts": p.counts,
            **({"masks": p.masks} if case["tree"] else {})}


def _own_append(case, s):
    from iris_b200 import serving
    serving.page_append(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_prompt(case, s):
    from iris_b200 import serving
    qd, kd = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    q, k, v = s["qkv"][:, :qd], s["qkv"][:, qd:qd + kd], s["qkv"][:, qd + kd:]
    return serving.prompt_attention(q, k, v, s["offsets"], s["longest"], heads=case["heads"], kv_heads=case["kv_heads"],
                                    scale_q32=_scale(case), window=case["window"])


def _own_tree(case, s):
    from iris_b200 import serving
    return serving.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["held"], s["offsets"], s["masks"],
                                  s["nodes"], s["longest"], heads=case["heads"], kv_heads=case["kv_heads"],
                                  scale_q32=_scale(case), window=case["window"], positions=s["positions"])


def _own_accept(case, s):
    from iris_b200 import serving
    a = serving.tree_accept(s["tokens"], s["parents"], s["picks"], s["offsets"], s["held"], s["table"], MAX_NODES,
                            k_pages=s["k_pages"], v_pages=s["v_pages"])
    return {"path": a.path, "accepted": a.accepted, "next": a.next, "held": a.held,
            "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---- plain forms ----------------------------------------------------------------

def _ancestors(parents, request, local, requests, nodes):
    """[requests][nodes][nodes]: whether column j is row i or one of its ancestors (a closure by repeated squaring)."""
    m = torch.eye(nodes, device=parents.device).repeat(requests, 1, 1)
    below = parents >= 0
    m[request[below], local[below], parents[below].long()] = 1.0

    def twice(x):
        return (x @ x > 0).float()

    return twice(twice(twice(twice(twice(twice(m)))))) > 0


def _rows(offsets, tokens):
    """The request of each packed row, and its place in it."""
    at = torch.arange(tokens, device=offsets.device)
    request = torch.searchsorted(offsets[1:].contiguous().long(), at, right=True)
    return request, at - offsets.long()[request]


def _plain_plan(case, s):
    held, fresh, table, free = s["held"].long(), s["fresh"].long(), s["table"], s["free"]
    offsets = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)])
    request, local = _rows(offsets, s["tokens"])
    before, after = (held + PAGE - 1) // PAGE, (held + fresh + PAGE - 1) // PAGE
    taken = (after - before).cumsum(0)
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    new = (column >= before[:, None]) & (column < after[:, None])
    which = (taken - (after - before))[:, None] + column - before[:, None]
    table.copy_(torch.where(new, free[which.clamp(0, free.numel() - 1)], table))
    at = held[request] + local
    slots = table[request, at // PAGE].long() * PAGE + at % PAGE
    counts = torch.stack([offsets[-1], taken[-1], offsets[-1] * 0, offsets[-1] * 0]).int()
    out = {"offsets": offsets.int(), "slots": slots, "positions": at.int(), "table": table, "counts": counts}
    if case["tree"]:
        anc = _ancestors(s["parents"], request, local, held.numel(), MAX_NODES)[request, local]
        out["positions"] = (held[request] + anc.sum(1) - 1).int()
        out["masks"] = (anc.long() << torch.arange(MAX_NODES, device=anc.device)).sum(1)
    return out


def _plain_append(case, s):
    kept = s["slots"] >= 0
    to = s["slots"][kept]
    s["k_pages"].view(-1, case["width"])[to] = s["k"][kept]
    s["v_pages"].view(-1, case["width"])[to] = s["v"][kept]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _shift_even(x, n):
    """x / 2^n to nearest, ties to even."""
    low, half = x & ((1 << n) - 1), 1 << (n - 1)
    f = x >> n
    return f + ((low > half) | ((low == half) & (f & 1 == 1)))


def _divide_even(n, d):
    """n / d to nearest, ties to even, both at least 0."""
    q = n // d
    r = n - q * d
    other = d - r
    return q + ((r > other) | ((r == other) & (q & 1 == 1)))


def _products(a, b):
    """sum over the last axis of a[..., m, :] b[..., n, :], modulo 2^64: in halves of 16 bits, exact in double."""
    b = b.transpose(-1, -2)
    ah, al, bh, bl = (a >> 16).double(), (a & 0xFFFF).double(), (b >> 16).double(), (b & 0xFFFF).double()
    out = (ah @ bh).long() << 32
    out += (ah @ bl + al @ bh).long() << 16
    out += (al @ bl).long()
    return out


def _scores(sums, scale):
    if scale:
        low = sums & 0xFFFFFFFF
        low = ((low >> 16) * scale + ((low & 0xFFFF) * scale >> 16)) >> 16
        sums = (sums >> 32) * scale + low
    return _shift_even(sums, 16).clamp(-2**31, 2**31 - 1)


def _exponentials(distance):
    """The terms of scores `distance` (at least 0) below the maximum."""
    ln2 = 2977044472
    x = distance.clamp(max=1 << 20) << 16
    k = x // ln2
    r = x - k * ln2
    del x

    def times_r(p):
        return _shift_even(p * r, 32)

    r2 = times_r(r)
    e = (1 << 32) - r + _divide_even(r2, 2)
    r3 = times_r(r2)
    e -= _divide_even(r3, 6)
    r4 = times_r(r3)
    e += _divide_even(r4, 24)
    e -= _divide_even(times_r(r4), 120)
    del r, r2, r3, r4
    one = torch.ones_like(k)
    half = (one << k) >> 1
    low, f = e & ((one << k) - 1), e >> k
    del e
    f += (low > half) | ((low == half) & (f & 1 == 1) & (k > 0))
    return torch.where(distance >= 1 << 20, 0, f)


def _attend(q, k, v, seen, scale):
    """q [..., m, d], k and v [..., n, d], seen [..., m, n] -> int32 [..., m, d]."""
    s = _scores(_products(q, k), scale)
    s.masked_fill_(~seen, -2**62)
    top = s.amax(-1, keepdim=True)
    index = torch.arange(s.shape[-1], device=s.device, dtype=torch.int32)
    first = torch.where(s == top, index, 2**31 - 1).amin(-1, keepdim=True).long()
    e = _exponentials((top - s).clamp_(max=2**31 - 1))
    del s
    e *= seen
    total = e.sum(-1, keepdim=True)
    total[total == 0] = 1
    high = (e << 16) // total  # e 2^32 / total in two steps of 16 bits: total is at most 2^47
    e = ((e << 16) - high * total) << 16
    low = _divide_even(e, total)
    del e
    w = _shift_even((high << 16) + low, 16)
    del high, low
    some = seen.any(-1, keepdim=True).expand_as(first)
    w.scatter_add_(-1, first, torch.where(some, 65536 - w.sum(-1, keepdim=True), 0))
    w = w.double()
    sums = ((w @ (v >> 16).double()).long() << 16) + (w @ (v & 0xFFFF).double()).long()
    return _shift_even(sums, 16).clamp(-2**31, 2**31 - 1).int()


def _plain_prompt(case, s):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    n = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([H * D, K * D, K * D], 1)
    request, at = _rows(s["offsets"], n)
    seen = (request[:, None] == request[None, :]) & (at[:, None] >= at[None, :])
    if case["window"]:
        seen &= at[:, None] - at[None, :] < case["window"]
    q = q.reshape(n, K, H // K, D).permute(1, 2, 0, 3)
    k, v = (x.reshape(n, K, D).transpose(0, 1)[:, None] for x in (k, v))
    return _attend(q, k, v, seen, _scale(case)).permute(2, 0, 1, 3).reshape(n, H * D)


def _plain_tree(case, s):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    table, held, rows = s["table"].clamp(min=0).long(), s["held"].long(), s["q"].shape[0]
    R, keys, T = table.shape[0], table.shape[1] * PAGE, s["nodes"]
    request, local = _rows(s["offsets"], rows)
    k, v = (x[table].view(R, keys, K, D).transpose(1, 2) for x in (s["k_pages"], s["v_pages"]))
    q = torch.zeros((R, T, H * D), dtype=torch.int32, device=k.device)
    q[request, local] = s["q"]
    q = q.view(R, T, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(R, K, H // K * T, D)
    mask, position = (torch.zeros((R, T), dtype=torch.int64, device=k.device) for _ in range(2))
    mask[request, local], position[request, local] = s["masks"], s["positions"].long()
    at = torch.arange(keys, device=k.device)[None, :]
    node = (at - held[:, None]).clamp(0, 63)
    cached = at < held[:, None]
    seen = cached[:, None, :] | ((mask[:, :, None] >> node[:, None, :] & 1 == 1) & (at - held[:, None] < T)[:, None, :])
    if case["window"]:
        where = torch.where(cached, at, position.gather(1, node.clamp(max=T - 1)))
        seen &= where[:, None, :] + case["window"] > position[:, :, None]
    seen = seen[:, None, None].expand(R, 1, H // K, T, keys).reshape(R, 1, H // K * T, keys)
    out = _attend(q, k, v, seen, _scale(case)).view(R, K, H // K, T, D).permute(0, 3, 1, 2, 4).reshape(R, T, H * D)
    return out[request, local]


def _plain_accept(case, s):
    held, offsets, R = s["held"].long(), s["offsets"], s["held"].numel()
    request, local = _rows(offsets, s["tokens"].numel())
    up, start = s["parents"].long(), offsets.long()[request]
    fits = (up >= 0) & (s["tokens"] == s["picks"][start + up.clamp(min=0)])
    # of the children that fit, the one of the lowest index
    node = torch.full((R, MAX_NODES), -1, dtype=torch.int64, device=up.device)
    node[request, local] = torch.where(fits, up, -1)
    earlier = torch.ones((MAX_NODES, MAX_NODES), dtype=torch.bool, device=up.device).tril(-1)
    same = (node[:, :, None] == node[:, None, :]) & earlier
    good = (node >= 0) & ~same.any(2)
    good[:, 0] = True
    anc = _ancestors(s["parents"], request, local, R, MAX_NODES)
    real = torch.zeros((R, MAX_NODES), dtype=torch.bool, device=up.device)
    real[request, local] = True
    taken = (good[:, None, :] | ~anc).all(2) & real
    accepted = taken.sum(1)
    rank = taken.cumsum(1) - 1
    path = torch.full((R, MAX_NODES + 1), -1, dtype=torch.int32, device=up.device)
    path.scatter_(1, torch.where(taken, rank, MAX_NODES), torch.arange(MAX_NODES, device=up.device, dtype=torch.int32).expand(R, -1))
    path = path[:, :MAX_NODES].contiguous()
    path.masked_fill_(torch.arange(MAX_NODES, device=up.device) >= accepted[:, None], -1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])[:, 0].long()
    follow = torch.where(accepted > 0, s["picks"][(offsets.long()[:-1] + last).clamp(0, s["picks"].numel() - 1)], -1)
    r, j = (path >= 0).nonzero(as_tuple=True)

    def slot(at):
        return s["table"][r, at // PAGE].long() * PAGE + at % PAGE

    source, target = slot(held[r] + path[r, j].long()), slot(held[r] + j)
    for_layers = (case["layers"], -1, case["width"])
    k, v = s["k_pages"].view(for_layers), s["v_pages"].view(for_layers)
    k[:, target], v[:, target] = k[:, source], v[:, source]
    return {"path": path, "accepted": accepted.int(), "next": follow.int(), "held": (held + accepted).int(),
            "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---- from the definitions, on the host --------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](case, {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in s.items()})


def _exact_plan(case, s):
    held, fresh, free, table = s["held"].tolist(), s["fresh"].tolist(), s["free"].tolist(), s["table"].clone()
    offsets, slots, positions, masks, taken = [0], [], [], [], 0
    for r, (h, f) in enumerate(zip(held, fresh)):
        for column in range(_pages(h), _pages(h + f)):
            table[r, column] = free[taken]
            taken += 1
        row, seen = table[r].tolist(), []
        for i in range(f):
            slots.append(row[(h + i) // PAGE] * PAGE + (h + i) % PAGE)
            if case["tree"]:
                up = int(s["parents"][offsets[-1] + i])
                seen.append((seen[up] if up >= 0 else 0) | 1 << i)
                positions.append(h + bin(seen[-1]).count("1") - 1)
            else:
                positions.append(h + i)
        masks += [m - (1 << 64) if m >> 63 else m for m in seen]
        offsets.append(offsets[-1] + f)
    out = {"offsets": torch.tensor(offsets, dtype=torch.int32), "slots": torch.tensor(slots, dtype=torch.int64),
           "positions": torch.tensor(positions, dtype=torch.int32), "table": table,
           "counts": torch.tensor([offsets[-1], taken, 0, 0], dtype=torch.int32)}
    if case["tree"]:
        out["masks"] = torch.tensor(masks, dtype=torch.int64)
    return out


def _exact_append(case, s):
    for i, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            s["k_pages"].view(-1, case["width"])[slot] = s["k"][i]
            s["v_pages"].view(-1, case["width"])[slot] = s["v"][i]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _exact_accept(case, s):
    if case["layers"] * case["requests"] * case["nodes"] > 20000:
        return None
    offsets, held = s["offsets"].tolist(), s["held"].tolist()
    layers, width = case["layers"], case["width"]
    k, v = s["k_pages"].view(layers, -1, width), s["v_pages"].view(layers, -1, width)
    paths, follow = [], []
    for r, h in enumerate(held):
        a, b = offsets[r], offsets[r + 1]
        path = _walk(s["parents"][a:b].tolist(), s["tokens"][a:b].tolist(), s["picks"][a:b].tolist())
        for j, i in enumerate(path):
            (x, y) = (int(s["table"][r, (h + n) // PAGE]) * PAGE + (h + n) % PAGE for n in (i, j))
            k[:, y], v[:, y] = k[:, x].clone(), v[:, x].clone()
        follow.append(int(s["picks"][a + path[-1]]))
        paths.append(path)
    return {"path": torch.tensor([p + [-1] * (MAX_NODES - len(p)) for p in paths], dtype=torch.int32),
            "accepted": torch.tensor([len(p) for p in paths], dtype=torch.int32), "next": torch.tensor(follow, dtype=torch.int32),
            "held": torch.tensor([h + len(p) for h, p in zip(held, paths)], dtype=torch.int32),
            "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _exact_row(q, k, v, scale):
    """One query against the keys that it sees, in Python's and numpy's 64-bit integers."""
    import numpy as np
    sums = (k * q).sum(1)  # wraps at 64 bits
    if scale:
        sums = np.array([(int(x) * scale) >> 32 for x in sums], dtype=np.int64)
    s = np.clip(_exact_half_even(sums, np.int64(16)), -2**31, 2**31 - 1)
    top = int(s.max())
    at = int((s == top).argmax())
    d = np.minimum(top - s, 2**31 - 1)
    near = d < 1 << 20
    x = np.where(near, d, 0).astype(np.int64) << 16
    turns, r = np.divmod(x, np.int64(2977044472))
    powers = [r]
    for _ in range(4):
        powers.append(_exact_half_even(powers[-1] * r, np.int64(32)))
    e = (1 << 32) - r
    for sign, p, n in ((1, powers[1], 2), (-1, powers[2], 6), (1, powers[3], 24), (-1, powers[4], 120)):
        a, b = np.divmod(p, n)
        e = e + sign * (a + ((2 * b > n) | ((2 * b == n) & (a % 2 == 1))))
    e = np.where(near, np.where(turns > 0, _exact_half_even(e, np.maximum(turns, 1)), e), 0)
    total = int(e.sum())
    w = np.zeros(len(e), dtype=np.int64)
    for i in np.nonzero(e)[0]:
        n, rest = divmod(int(e[i]) << 32, total)
        n += 2 * rest > total or (2 * rest == total and n % 2 == 1)
        w[i] = (n >> 16) + ((n & 0xFFFF) > 0x8000 or ((n & 0xFFFF) == 0x8000 and (n >> 16) % 2 == 1))
    w[at] += 65536 - int(w.sum())
    return np.clip(_exact_half_even((w[:, None] * v).sum(0), np.int64(16)), -2**31, 2**31 - 1)


def _exact_half_even(x, n):
    import numpy as np
    f = x >> n
    rest = x - (f << n)
    half = np.int64(1) << (n - 1)
    return f + ((rest > half) | ((rest == half) & (f % 2 == 1)))


def _exact_prompt(case, s):
    import numpy as np
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    lengths = _numbers(case["lengths"])
    if H * sum(n * min(n, case["window"] or n) for n in lengths) > 4_000_000:
        return None
    x = s["qkv"].numpy().astype(np.int64)
    q, k, v = (y.reshape(len(x), -1, D) for y in np.split(x, [H * D, (H + K) * D], 1))
    out = np.zeros((len(x), H, D), dtype=np.int32)
    for a, n in zip(_offsets(lengths), lengths):
        for i in range(n):
            lo = max(0, i + 1 - case["window"]) if case["window"] else 0
            for h in range(H):
                seen = slice(a + lo, a + i + 1), h * K // H
                out[a + i, h] = _exact_row(q[a + i, h], k[seen], v[seen], _scale(case))
    return torch.from_numpy(out.reshape(len(x), H * D))


def _exact_tree(case, s):
    import numpy as np
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    held, nodes = _numbers(case["held"]), _numbers(case["nodes"])
    if H * sum((h + n) * n for h, n in zip(held, nodes)) > 4_000_000:
        return None
    q = s["q"].numpy().astype(np.int64).reshape(-1, H, D)
    k, v = (x.numpy().reshape(-1, PAGE, K, D) for x in (s["k_pages"], s["v_pages"]))
    out = np.zeros(q.shape, dtype=np.int32)
    for r, (a, h, n) in enumerate(zip(_offsets(nodes), held, nodes)):
        pages = s["table"][r, :_pages(h + n)].numpy()
        kr, vr = (x[pages].reshape(-1, K, D)[:h + n].astype(np.int64) for x in (k, v))
        position = s["positions"][a:a + n].tolist()
        for i in range(n):
            mask = int(s["masks"][a + i])
            low = max(0, position[i] + 1 - case["window"]) if case["window"] else 0
            seen = list(range(low, h)) + [h + j for j in range(n) if mask >> j & 1 and position[j] >= low]
            for head in range(H):
                g = head * K // H
                if seen:
                    out[a + i, head] = _exact_row(q[a + i, head], kr[seen, g], vr[seen, g], _scale(case))
    return torch.from_numpy(out.reshape(-1, H * D))
