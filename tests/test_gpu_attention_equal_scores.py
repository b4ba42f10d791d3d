"""Prefill attention over many equal scores: 724 or more equal weights round up
to more than 1.0 together, and what is left for the first maximum is negative
(attention_softmax, ops.rs:233-276)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    from iris_b200 import build
    from oracle import oracle
    build.build()
    oracle.build()


@pytest.mark.parametrize("start,m", [(0, 40), (700, 64), (800, 33), (1100, 100), (3000, 40)])
def test_equal_scores_equal_the_oracle(start, m):
    """Keys of zeros (a key projection of zero weights): every score is 0, the first position takes the residual."""
    from iris_b200.model import DeviceModel, synth_host_weights
    from iris_b200.shapes import MistralConfig
    from oracle.models import OracleModel
    cfg = MistralConfig("mistral-d128-small", layers=1, hidden=256, ffn=512, heads=4, kv_heads=1, head_dim=128,
                        vocab=512, rope_base=1_000_000, max_positions=16384, tied=True)
    w = synth_host_weights(cfg, 0xE9)
    w["W_K", 0].reshape(-1, 34)[:, 2:] = 0  # the blocks' values, not their scales
    rng = np.random.default_rng(start + m)
    rows = rng.integers(-(4 << 16), 4 << 16, size=(m, cfg.hidden)).astype(np.int32)
    kvd = cfg.kv_heads * cfg.head_dim
    prior_k = np.zeros((start, kvd), np.int32)
    prior_v = rng.integers(-(1 << 22), 1 << 22, size=(start, kvd)).astype(np.int32)
    dm = DeviceModel(cfg, weights=w)
    got = dm.layer_range(0, rows, start, prior_k, prior_v)
    assert dm.attention_ranges() == (1, 0)  # on the tensor cores
    dm.close()
    want = OracleModel(cfg, w).mistral_layer_range(0, rows, start, prior_k, prior_v)
    for g, wnt, what in zip(got, want, ("rows", "k", "v")):
        assert np.array_equal(g, wnt), what
