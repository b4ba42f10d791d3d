"""Serving many requests over one paged K/V cache: a step's block tables and
slot map, packed prompts, drafted trees and their acceptance.

The operators take CUDA tensors (int32 Q16.16 rows, as every activation of the
library) and run in libiris_b200.so on torch's current stream, asynchronously
and without host synchronisation; outputs and scratch come from torch's
allocator. Their arithmetic is the decode loop's, so a token verified in a
drafted tree, or a prompt row packed among others, has the values that
decoding it alone gives, bit for bit. include/iris_b200.h (section 6) states
each operator's contract; a refused argument raises IrisError (or ValueError
where a tensor has the wrong type, shape or device).

One step of a drafted decode:

    plan = page_plan(held, fresh, table, free_pages, page_size, tokens, parents=parents)
    ... q, k, v rows of the drafted tokens at plan.positions ...
    page_append(k, v, plan.slots, k_pages, v_pages)            # each layer
    ctx = tree_attention(q, k_pages, v_pages, plan.table, held, plan.offsets, plan.masks, ...)
    ... picks = the model's first-maximum token after each node ...
    done = tree_accept(tokens, parents, picks, plan.offsets, held, plan.table, nodes,
                       k_pages=all_k, v_pages=all_v)           # all layers at once
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check, lib

TREE_NODES = 64  # drafted nodes a request
U32 = 1 << 32


class PagePlan(NamedTuple):
    """The bookkeeping of a step (page_plan). faults() waits for the device."""
    offsets: torch.Tensor    # [requests + 1] packed rows of each request
    slots: torch.Tensor      # [tokens] int64 pool rows, -1: none
    positions: torch.Tensor  # [tokens]
    table: torch.Tensor      # [requests][width], the one passed in
    counts: torch.Tensor     # {tokens, pages taken, tokens left out, faults}
    masks: Optional[torch.Tensor]  # [tokens] int64, with parents

    def faults(self) -> int:
        """PLAN_* bits of this plan (0: the pages, the table and the rows sufficed)."""
        return int(self.counts[3])


class Accepted(NamedTuple):
    path: torch.Tensor      # [requests][path_width] accepted nodes, -1 after the last
    accepted: torch.Tensor  # [requests]
    next: torch.Tensor      # [requests] the token after the last accepted one
    held: torch.Tensor      # [requests] cached tokens now


def _refuse(x: torch.Tensor, name: str, dtype: torch.dtype, dim: int, what: str) -> None:
    raise ValueError(f"{name}: a CUDA tensor of {dtype} with {dim} axes, {what}, on the device of the call's first "
                     f"tensor, is needed; got {x.dtype} {tuple(x.shape)} on {x.device} with strides {x.stride()}")


def _rows(x: torch.Tensor, name: str, dev: int) -> int:
    """The address of int32 rows on device `dev` whose last axis is dense (rows may lie apart)."""
    if (x.dtype != torch.int32 or dev < 0 or x.get_device() != dev or x.dim() != 2
            or (x.stride(1) != 1 and x.numel())):
        _refuse(x, name, torch.int32, 2, "the last one dense")
    return x.data_ptr()


def _dense(x: torch.Tensor, name: str, dev: int, dtype: torch.dtype = torch.int32, dim: int = 1) -> int:
    """The address of a contiguous tensor on device `dev`."""
    if x.dtype != dtype or dev < 0 or x.get_device() != dev or x.dim() != dim or not x.is_contiguous():
        _refuse(x, name, dtype, dim, "contiguous")
    return x.data_ptr()


def _stride(x: torch.Tensor, rows: int, width: int) -> int:
    """The values between two rows; of a single row torch may give any."""
    return x.stride(0) if rows != 1 else width


def _same(count: int, want: int, name: str) -> None:
    if count != want:
        raise ValueError(f"{name}: {count} entries, expected {want}")


def _ranges(**values: int) -> None:
    """Refuses what is no 32-bit count (ctypes would cut it to one)."""
    for name, value in values.items():
        if not 0 <= value < U32:
            raise ValueError(f"{name}: {value} is not between 0 and 2^32 - 1")


def _stream(index: int) -> int:
    """torch's current stream on the tensors' device, which has to be the current one."""
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"tensors are on cuda:{index}, but cuda:{torch.cuda.current_device()} is the current device")
    return torch._C._cuda_getCurrentRawStream(index)


def page_plan(held: torch.Tensor, fresh: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page_size: int,
              tokens: int, parents: Optional[torch.Tensor] = None) -> PagePlan:
    """Block tables and slot map of a step: request r has held[r] cached tokens
    and brings fresh[r]. New pages are taken from free_pages in order and
    written into `table` [requests][width]. `tokens`: rows of the outputs (at
    least the fresh tokens). With `parents` (each drafted node's parent in its
    request, -1 for a root) the plan has the nodes' visibility masks and their
    positions count ancestors only."""
    dev = held.get_device()
    ph, pf = _dense(held, "held", dev), _dense(fresh, "fresh", dev)
    pt, pp = _dense(table, "table", dev, dim=2), _dense(free_pages, "free_pages", dev)
    requests, width, n_free = held.numel(), table.shape[1], free_pages.numel()
    if not (0 <= page_size < U32 and 0 <= tokens < U32):
        _ranges(page_size=page_size, tokens=tokens)
    _same(fresh.numel(), requests, "fresh")
    _same(table.shape[0], requests, "table")
    masks, pa, pm = None, None, None
    if parents is not None:
        if parents.numel() < tokens:
            raise ValueError(f"parents: {parents.numel()} entries, expected {tokens}")
        pa = _dense(parents, "parents", dev)
    counts, offsets, positions = held.new_empty(4), held.new_empty(requests + 1), held.new_empty(tokens)
    slots = torch.empty(tokens, dtype=torch.int64, device=held.device)
    if parents is not None:
        masks = slots.new_empty(tokens)
        pm = masks.data_ptr()
    check(lib().iris_page_plan(ph, pf, requests, page_size, pt, width, pp, n_free, pa, tokens, offsets.data_ptr(),
                               slots.data_ptr(), positions.data_ptr(), pm, counts.data_ptr(), _stream(dev)),
          "iris_page_plan")
    return PagePlan(offsets, slots, positions, table, counts, masks)


def page_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor,
                v_pages: torch.Tensor) -> None:
    """K and V rows [tokens][kv_dim] into the pools [pages][page_size][kv_dim]
    at their slots; a slot outside the pools (-1) skips its row."""
    dev = k.get_device()
    pk, pv, ps = _rows(k, "k", dev), _rows(v, "v", dev), _dense(slots, "slots", dev, torch.int64)
    ck, cv = _dense(k_pages, "k_pages", dev, dim=3), _dense(v_pages, "v_pages", dev, dim=3)
    tokens, kv_dim = k.shape
    if v.shape != k.shape or k_pages.shape != v_pages.shape or k_pages.shape[2] != kv_dim:
        raise ValueError(f"rows {tuple(k.shape)}, {tuple(v.shape)} and pools {tuple(k_pages.shape)}, "
                         f"{tuple(v_pages.shape)} do not match")
    _same(slots.numel(), tokens, "slots")
    check(lib().iris_page_append(pk, pv, _stride(k, tokens, kv_dim), _stride(v, tokens, kv_dim), tokens, kv_dim, ps, ck,
                                 cv, k_pages.shape[0] * k_pages.shape[1], _stream(dev)), "iris_page_append")


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, longest: int, *,
                     heads: int, kv_heads: int, scale_q32: int = 0, window: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts: q [tokens][heads * head_dim], k and v
    [tokens][kv_heads * head_dim] (rows may be parts of a fused q|k|v row);
    request r's rows are offsets[r] .. offsets[r + 1] - 1, the longest request
    at most `longest` rows. scale_q32 0: unscaled scores (gemma-dense). Rows past
    the last request's are left as `out` has them (undefined without it)."""
    dev = q.get_device()
    pq, pk, pv, po = _rows(q, "q", dev), _rows(k, "k", dev), _rows(v, "v", dev), _dense(offsets, "offsets", dev)
    tokens, requests = q.shape[0], offsets.numel() - 1
    if not (0 <= requests and 0 <= longest < U32 and 0 <= heads < U32 and 0 <= kv_heads < U32 and 0 <= window < U32
            and 0 <= scale_q32 < U32):
        _ranges(requests=requests, longest=longest, heads=heads, kv_heads=kv_heads, window=window, scale_q32=scale_q32)
    if heads < 1 or kv_heads < 1 or q.shape[1] % heads:
        raise ValueError(f"q rows of {q.shape[1]} values are not {heads} heads")
    dim = q.shape[1] // heads
    if k.shape != (tokens, kv_heads * dim) or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not {tokens} rows of {kv_heads} heads of {dim}")
    if out is None:
        out = q.new_empty((tokens, heads * dim))
    elif out.shape != q.shape:
        raise ValueError(f"out: {tuple(out.shape)}, expected {tuple(q.shape)}")
    qd, kd = heads * dim, kv_heads * dim
    a = _lib.PromptAttention(pq, pk, pv, po, _rows(out, "out", dev), _stride(q, tokens, qd), _stride(k, tokens, kd),
                             _stride(v, tokens, kd), _stride(out, tokens, qd), requests, tokens, longest, heads,
                             kv_heads, dim, window, scale_q32)
    L, ref = lib(), C.byref(a)
    ws = _workspace(L.iris_prompt_attention_workspace(ref), q.device)
    check(L.iris_prompt_attention(ref, ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                                  _stream(dev)), "iris_prompt_attention")
    return out


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                   held: torch.Tensor, offsets: torch.Tensor, masks: torch.Tensor, nodes: int, longest: int, *,
                   heads: int, kv_heads: int, scale_q32: int = 0, window: int = 0,
                   positions: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of drafted nodes over the paged cache, their K/V appended
    already: q [rows][heads * head_dim], request r's nodes the rows offsets[r]
    .. offsets[r + 1] - 1 (at most `nodes` each), a node seeing the held[r]
    cached tokens and the nodes of its mask. `longest`: the most cached tokens
    and nodes a request has together. A node that sees nothing gives zeros; rows
    past the last request's nodes are left as `out` has them (undefined without it)."""
    dev = q.get_device()
    pq, ck, cv = _rows(q, "q", dev), _dense(k_pages, "k_pages", dev, dim=3), _dense(v_pages, "v_pages", dev, dim=3)
    pt, ph, po = _dense(table, "table", dev, dim=2), _dense(held, "held", dev), _dense(offsets, "offsets", dev)
    pm = _dense(masks, "masks", dev, torch.int64)
    pp = _dense(positions, "positions", dev) if positions is not None else None
    rows, requests = q.shape[0], held.numel()
    if not (0 <= nodes < U32 and 0 <= longest < U32 and 0 <= heads < U32 and 0 <= kv_heads < U32 and 0 <= window < U32
            and 0 <= scale_q32 < U32):
        _ranges(nodes=nodes, longest=longest, heads=heads, kv_heads=kv_heads, window=window, scale_q32=scale_q32)
    if heads < 1 or kv_heads < 1 or q.shape[1] % heads:
        raise ValueError(f"q rows of {q.shape[1]} values are not {heads} heads")
    dim = q.shape[1] // heads
    if k_pages.shape != v_pages.shape or k_pages.shape[2] != kv_heads * dim:
        raise ValueError(f"pools {tuple(k_pages.shape)}, {tuple(v_pages.shape)} do not hold {kv_heads} heads of {dim}")
    _same(table.shape[0], requests, "table")
    _same(offsets.numel(), requests + 1, "offsets")
    for x, name in ((masks, "masks"), (positions, "positions")):
        if x is not None and x.numel() < rows:
            raise ValueError(f"{name}: {x.numel()} entries, expected {rows}")
    if out is None:
        out = q.new_empty((rows, heads * dim))
    elif out.shape != q.shape:
        raise ValueError(f"out: {tuple(out.shape)}, expected {tuple(q.shape)}")
    a = _lib.TreeAttention(pq, ck, cv, pt, ph, po, pm, pp, _rows(out, "out", dev), _stride(q, rows, heads * dim),
                           _stride(out, rows, heads * dim), k_pages.shape[0], requests, rows, table.shape[1],
                           k_pages.shape[1], nodes, longest, heads, kv_heads, dim, window, scale_q32)
    L, ref = lib(), C.byref(a)
    ws = _workspace(L.iris_tree_attention_workspace(ref), q.device)
    check(L.iris_tree_attention(ref, ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                                _stream(dev)), "iris_tree_attention")
    return out


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, picks: torch.Tensor, offsets: torch.Tensor,
                held: torch.Tensor, table: torch.Tensor, path_width: int, *, k_pages: Optional[torch.Tensor] = None,
                v_pages: Optional[torch.Tensor] = None) -> Accepted:
    """The drafted nodes that greedy decoding accepts (from node 0, to the
    child that holds the pick, until none does) and, with pools
    [layers][pages][page_size][kv_dim], their K/V rows moved after the cached
    ones, in place, in every layer."""
    rows, requests = tokens.numel(), held.numel()
    dev = tokens.get_device()
    pt, pa, pk = _dense(tokens, "tokens", dev), _dense(parents, "parents", dev), _dense(picks, "picks", dev)
    po, ph, tb = _dense(offsets, "offsets", dev), _dense(held, "held", dev), _dense(table, "table", dev, dim=2)
    if not 0 <= path_width < U32:
        _ranges(path_width=path_width)
    _same(parents.numel(), rows, "parents")
    _same(picks.numel(), rows, "picks")
    _same(offsets.numel(), requests + 1, "offsets")
    _same(table.shape[0], requests, "table")
    layers, stride, pages, page, kv_dim, ck, cv = 0, 0, 0, 0, 0, None, None
    if k_pages is not None or v_pages is not None:
        if k_pages is None or v_pages is None or k_pages.shape != v_pages.shape:
            raise ValueError("k_pages and v_pages are given together, of one shape")
        ck, cv = _dense(k_pages, "k_pages", dev, dim=4), _dense(v_pages, "v_pages", dev, dim=4)
        layers, pages, page, kv_dim = k_pages.shape
        stride = pages * page * kv_dim
    accepted, after, now = held.new_empty(requests), held.new_empty(requests), held.new_empty(requests)
    path = held.new_empty((requests, path_width))
    check(lib().iris_tree_accept(pt, pa, pk, po, requests, rows, ph, path_width, path.data_ptr(), accepted.data_ptr(),
                                 after.data_ptr(), now.data_ptr(), tb, table.shape[1], page, ck, cv, layers, stride,
                                 pages, kv_dim, _stream(dev)), "iris_tree_accept")
    return Accepted(path, accepted, after, now)


def stall_check() -> None:
    """Waits for torch's current stream; raises IrisError if a kernel of the
    library gave up a bounded wait since the last check (its rows are then
    undefined)."""
    check(lib().iris_stall_check(torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())), "iris_stall_check")
