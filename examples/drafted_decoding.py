"""Drafted decoding of several requests over one paged K/V cache.

Packed prompts fill the cache, then every step drafts a small tree of tokens a
request, scores all nodes in one pass, keeps the path that greedy decoding
agrees with and drops the others. The tokens are those of decoding one by one:

    python examples/drafted_decoding.py --requests 6 --tokens 48

The model is a stand-in (integer rows from fixed random tables, exact in any
batch), the drafts are the right continuation with mistakes mixed in; the cache,
the attention and the acceptance are iris_b200.serving's.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from iris_b200 import serving  # noqa: E402
from iris_b200.shapes import attention_scale_q32  # noqa: E402

VOCAB, LAYERS, HEADS, KV_HEADS, DIM, PAGE = 64, 2, 8, 2, 64, 16


class Model:
    """q, k and v rows of a token at a position, and the token that follows a context row."""

    def __init__(self, seed: int, longest: int):
        g = torch.Generator().manual_seed(seed)

        def table(*shape: int) -> torch.Tensor:
            return (torch.randn(shape, generator=g) * 65536).int().cuda()

        self.width = (HEADS + 2 * KV_HEADS) * DIM
        self.token = table(LAYERS, VOCAB, self.width)
        self.place = table(LAYERS, longest, self.width)
        self.head = torch.randint(-8, 9, (HEADS * DIM, VOCAB), generator=g).double().cuda()

    def qkv(self, layer: int, tokens: torch.Tensor, positions: torch.Tensor, below: torch.Tensor) -> torch.Tensor:
        rows = self.token[layer][tokens.long()] + self.place[layer][positions.long()]
        rows[:, :HEADS * DIM] += below
        return rows

    def picks(self, rows: torch.Tensor) -> torch.Tensor:
        """The first maximum of each row's logits (integers below 2^53: doubles add them exactly)."""
        logits = rows.double() @ self.head
        first = logits == logits.max(1, keepdim=True).values
        return torch.where(first, torch.arange(VOCAB, device=rows.device), VOCAB).min(1).values.int()


class Cache:
    """Page pools for every layer, the requests' block tables and the pages nobody holds."""

    def __init__(self, requests: int, longest: int):
        self.width = -(-longest // PAGE)
        pages = requests * self.width
        shape = (LAYERS, pages, PAGE, KV_HEADS * DIM)
        self.k, self.v = (torch.zeros(shape, dtype=torch.int32, device="cuda") for _ in range(2))
        self.table = torch.full((requests, self.width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def plan(self, fresh: torch.Tensor, tokens: int, parents=None) -> serving.PagePlan:
        plan = serving.page_plan(self.held, fresh, self.table, self.free, PAGE, tokens, parents=parents)
        if plan.faults():
            raise RuntimeError(f"the step does not fit the cache (faults {plan.faults()})")
        self.free = self.free[int(plan.counts[1]):].contiguous()
        return plan

    def keep(self, held: torch.Tensor) -> None:
        """The requests' lengths now; pages past them are free again."""
        self.held = held
        unused = torch.arange(self.width, device="cuda")[None] >= ((held + PAGE - 1) // PAGE)[:, None]
        self.free = torch.cat([self.free, self.table[unused & (self.table >= 0)]])
        self.table[unused] = -1


def forward(model: Model, cache: Cache, tokens: torch.Tensor, plan: serving.PagePlan, longest: int, nodes: int) -> torch.Tensor:
    """Context rows of the step's tokens: drafted trees where the plan has masks (at most `nodes` a request), else prompts."""
    q_dim, kv_dim, scale = HEADS * DIM, KV_HEADS * DIM, attention_scale_q32(DIM)
    rows = torch.zeros((tokens.numel(), q_dim), dtype=torch.int32, device="cuda")
    for layer in range(LAYERS):
        q, k, v = model.qkv(layer, tokens, plan.positions, rows).split([q_dim, kv_dim, kv_dim], 1)
        serving.page_append(k, v, plan.slots, cache.k[layer], cache.v[layer])
        if plan.masks is None:
            rows = serving.prompt_attention(q, k, v, plan.offsets, longest, heads=HEADS, kv_heads=KV_HEADS,
                                            scale_q32=scale)
        else:
            rows = serving.tree_attention(q, cache.k[layer], cache.v[layer], plan.table, cache.held, plan.offsets,
                                          plan.masks, nodes, longest, heads=HEADS, kv_heads=KV_HEADS, scale_q32=scale)
    return rows


def draft(last: int, right: list[int], nodes: int, g: torch.Generator) -> tuple[list[int], list[int]]:
    """A tree of `nodes` tokens under `last`: the right continuation in part, wrong tokens beside it."""
    tokens, parents, tip = [last], [-1], 0
    for i in range(1, nodes):
        depth = i - 1 if tip == i - 1 else None  # the right path's next token, while it is unbroken
        if depth is not None and depth < len(right) and torch.rand((), generator=g) < 0.8:
            tokens.append(right[depth])
            parents.append(tip)
            tip = i
        else:
            tokens.append(int(torch.randint(VOCAB, (), generator=g)))
            parents.append(int(torch.randint(i, (), generator=g)))
    return tokens, parents


def decode(model: Model, prompts: list[list[int]], count: int, nodes: int, seed: int = 0, right=None) -> tuple[list[list[int]], int]:
    """`count` tokens after each prompt, and the steps they took: one node a
    request and step is plain decoding; more follow the drafts made from `right`."""
    g = torch.Generator().manual_seed(seed)
    longest = max(map(len, prompts)) + count + 2 * nodes
    cache = Cache(len(prompts), longest)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    lengths = ints([len(p) for p in prompts])
    plan = cache.plan(lengths, sum(map(len, prompts)))
    rows = forward(model, cache, ints(sum(prompts, [])), plan, max(map(len, prompts)), 0)
    cache.held = lengths
    out = [[t] for t in model.picks(rows[(plan.offsets[1:] - 1).long()]).tolist()]
    steps = 0
    while min(map(len, out)) < count:
        steps += 1
        trees = [draft(o[-1], right[r][len(o):] if right else [], nodes, g) if len(o) < count else ([], [])
                 for r, o in enumerate(out)]  # a request that is done brings no more nodes
        tokens, parents = (ints(sum((t[i] for t in trees), [])) for i in (0, 1))
        plan = cache.plan(ints([len(t[0]) for t in trees]), tokens.numel(), parents)
        rows = forward(model, cache, tokens, plan, longest, nodes)
        done = serving.tree_accept(tokens, parents, model.picks(rows), plan.offsets, cache.held, cache.table, nodes,
                                   k_pages=cache.k, v_pages=cache.v)
        cache.keep(done.held)
        for r, (path, after) in enumerate(zip(done.path.tolist(), done.next.tolist())):
            if trees[r][0]:
                out[r] += [trees[r][0][i] for i in path[1:] if i >= 0] + [after]
    serving.stall_check()
    return [o[:count] for o in out], steps


def run(requests: int, count: int, nodes: int, seed: int = 0) -> tuple[list[list[int]], list[list[int]], int, int]:
    """(plain tokens, drafted tokens, plain steps, drafted steps)."""
    g = torch.Generator().manual_seed(seed + 1)
    prompts = [torch.randint(VOCAB, (int(torch.randint(1, 40, (), generator=g)),), generator=g).tolist()
               for _ in range(requests)]
    model = Model(seed, 40 + count + 2 * nodes)
    plain, plain_steps = decode(model, prompts, count, 1)
    drafted, steps = decode(model, prompts, count, nodes, seed, plain)
    return plain, drafted, plain_steps, steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--nodes", type=int, default=12, help="drafted nodes a request and step (64 at most)")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    plain, drafted, plain_steps, steps = run(a.requests, a.tokens, a.nodes, a.seed)
    print(f"one by one: {plain_steps} steps; drafted: {steps} steps; the same tokens: {plain == drafted}")
    if plain != drafted:
        raise SystemExit(1)


if __name__ == "__main__":
    main()
