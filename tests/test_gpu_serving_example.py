"""The drafted decoding example: the serving operators as a user runs them."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,count,nodes", [(1, 5, 1), (5, 40, 12), (3, 70, 64)])
def test_drafted_tokens_are_those_of_plain_decoding(requests, count, nodes):
    from iris_b200 import build
    build.build()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "drafted_decoding.py")
    spec = importlib.util.spec_from_file_location("drafted_decoding", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    plain, drafted, plain_steps, steps = example.run(requests, count, nodes)
    assert drafted == plain and all(len(t) == count for t in plain)
    assert plain_steps == count - 1 and (nodes == 1 or steps < plain_steps)
    assert len({tuple(t) for t in plain}) == requests  # each request has its own continuation
