"""What the serving operators refuse, before anything is launched (no GPU):
through the C ABI with addresses that are never read, and in the Python
wrappers' own checks."""
import ctypes as C

import pytest

A = 1 << 20  # a 16-byte aligned address that nothing reads: every call here is refused first


@pytest.fixture(scope="module")
def lib():
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib
    return _lib


def prompt(lib, **changes):
    a = dict(q=A, k=A, v=A, offsets=A, out=A, q_stride=512, k_stride=256, v_stride=256, out_stride=512, requests=1,
             tokens=8, longest=8, heads=4, kv_heads=2, head_dim=128, window=0, scale_q32=1)
    a.update(changes)
    return lib.PromptAttention(**a)


def tree(lib, **changes):
    a = dict(q=A, k_pages=A, v_pages=A, table=A, held=A, offsets=A, masks=A, positions=None, out=A, q_stride=512,
             out_stride=512, pages=4, requests=1, rows=3, width=2, page_size=16, nodes=3, longest=20, heads=4,
             kv_heads=2, head_dim=128, window=0, scale_q32=1)
    a.update(changes)
    return lib.TreeAttention(**a)


@pytest.mark.parametrize("changes", [
    dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(head_dim=0), dict(head_dim=130), dict(head_dim=260),
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(offsets=None), dict(q=A + 4), dict(out=A + 8),
    dict(q_stride=508), dict(k_stride=252), dict(v_stride=258), dict(out_stride=514), dict(requests=0),
    dict(longest=0), dict(tokens=1 << 31), dict(heads=65536, kv_heads=65536, head_dim=4)])
def test_prompt_attention_refuses(lib, changes):
    a = prompt(lib, **changes)
    assert lib.lib().iris_prompt_attention(C.byref(a), None, 0, None) == lib.IRIS_EINVAL
    assert lib.lib().iris_prompt_attention_workspace(C.byref(a)) == 0


@pytest.mark.parametrize("changes", [
    dict(heads=0), dict(kv_heads=3), dict(head_dim=6), dict(head_dim=512), dict(q=None), dict(k_pages=None),
    dict(v_pages=A + 12), dict(table=None), dict(held=None), dict(offsets=None), dict(masks=None), dict(out=None),
    dict(window=8), dict(nodes=0), dict(nodes=65), dict(page_size=0), dict(width=0), dict(longest=33),
    dict(q_stride=510), dict(out_stride=4), dict(requests=0), dict(rows=1 << 31), dict(pages=1 << 32)])
def test_tree_attention_refuses(lib, changes):
    a = tree(lib, **changes)
    assert lib.lib().iris_tree_attention(C.byref(a), None, 0, None) == lib.IRIS_EINVAL
    assert lib.lib().iris_tree_attention_workspace(C.byref(a)) == 0


def test_no_rows_are_no_work(lib):
    L = lib.lib()
    assert L.iris_prompt_attention(C.byref(prompt(lib, tokens=0, q=None)), None, 0, None) == 0
    assert L.iris_tree_attention(C.byref(tree(lib, rows=0, q=None)), None, 0, None) == 0
    assert L.iris_page_append(None, None, 0, 0, 0, 64, None, None, None, 16, None) == 0
    assert L.iris_tree_accept(None, None, None, None, 0, 0, None, 64, None, None, None, None, None, 0, 16, None, None,
                              0, 0, 0, 0, None) == 0
    assert L.iris_prompt_attention(None, None, 0, None) == lib.IRIS_EINVAL
    assert L.iris_tree_attention(None, None, 0, None) == lib.IRIS_EINVAL


def test_page_plan_refuses(lib):
    L = lib.lib()

    def plan(held=A, fresh=A, requests=2, page=16, table=A, width=3, free=A, n_free=4, parents=None, tokens=5, offsets=A,
             slots=A, positions=A, masks=None, counts=A):
        return L.iris_page_plan(held, fresh, requests, page, table, width, free, n_free, parents, tokens, offsets, slots,
                                positions, masks, counts, None)

    for bad in (dict(held=None), dict(fresh=None), dict(requests=16385), dict(page=0), dict(page=(1 << 20) + 1),
                dict(table=None), dict(free=None), dict(tokens=1 << 31), dict(offsets=None), dict(slots=None),
                dict(positions=None), dict(counts=None), dict(parents=A), dict(masks=A)):
        assert plan(**bad) == lib.IRIS_EINVAL, bad


def test_page_append_refuses(lib):
    L = lib.lib()

    def append(k=A, v=A, ks=64, vs=64, tokens=3, dim=64, slots=A, kp=A, vp=A, rows=32):
        return L.iris_page_append(k, v, ks, vs, tokens, dim, slots, kp, vp, rows, None)

    for bad in (dict(k=None), dict(v=None), dict(k=A + 4), dict(ks=60), dict(vs=66), dict(dim=0), dict(dim=62),
                dict(slots=None), dict(kp=None), dict(vp=A + 8), dict(tokens=1 << 31), dict(rows=1 << 41)):
        assert append(**bad) == lib.IRIS_EINVAL, bad


def test_tree_accept_refuses(lib):
    L = lib.lib()

    def accept(tokens=A, parents=A, picks=A, offsets=A, requests=2, rows=5, held=A, width=64, path=A, accepted=A, nxt=A,
               held_out=A, table=A, cols=3, page=16, k=A, v=A, layers=2, stride=4 * 16 * 64, pages=4, dim=64):
        return L.iris_tree_accept(tokens, parents, picks, offsets, requests, rows, held, width, path, accepted, nxt,
                                  held_out, table, cols, page, k, v, layers, stride, pages, dim, None)

    for bad in (dict(tokens=None), dict(parents=None), dict(picks=None), dict(offsets=None), dict(held=None),
                dict(width=0), dict(width=65), dict(path=None), dict(accepted=None), dict(nxt=None), dict(held_out=None),
                dict(table=None), dict(page=0), dict(k=None), dict(v=None), dict(k=A + 4), dict(layers=0),
                dict(layers=65536), dict(stride=4 * 16 * 64 - 4), dict(stride=4 * 16 * 64 + 2), dict(dim=0), dict(dim=62),
                dict(rows=1 << 31)):
        assert accept(**bad) == lib.IRIS_EINVAL, bad


def test_the_wrappers_refuse_what_is_no_cuda_row(lib):
    import torch
    from iris_b200 import serving as S
    host = torch.zeros((3, 64), dtype=torch.int32)
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.prompt_attention(host, host, host, ints, 3, heads=1, kv_heads=1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.page_append(host, host, ints.long(), host[None], host[None])
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.page_plan(ints, ints, host, ints, 16, 3)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.tree_accept(ints, ints, ints, ints, ints, host, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.tree_attention(host, host[None], host[None], host, ints, ints, ints.long(), 3, 3, heads=1, kv_heads=1)
