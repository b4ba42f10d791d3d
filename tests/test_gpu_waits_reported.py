"""A wait that gave up is reported to each that asks: a session's pass and the
serving check each say so once, whichever comes first."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    from iris_b200 import build
    build.build()
    from iris_b200 import _lib
    lib = _lib.lib()
    assert lib.q8gpu_init() == 0
    return lib


def stalled(call):
    from iris_b200 import _lib
    try:
        call()
    except _lib.IrisError as e:
        assert e.code == _lib.IRIS_ESTALL
        return True
    return False


@pytest.mark.parametrize("first", ["session", "serving"])
def test_a_session_and_the_serving_check_each_report_a_give_up_once(L, first):
    from iris_b200 import _lib, serving
    from iris_b200.model import DeviceModel, synth_host_weights
    from iris_b200.shapes import MistralConfig
    cfg = MistralConfig("mistral-d128-small", layers=1, hidden=256, ffn=512, heads=4, kv_heads=1, head_dim=128,
                        vocab=512, rope_base=1_000_000, max_positions=16384, tied=True)
    dm = DeviceModel(cfg, weights=synth_host_weights(cfg, 3))

    def generate():
        session = dm.session(64)
        try:
            return session.generate([1, 2, 3], 4)
        finally:
            session.close()

    want = generate()
    assert not stalled(serving.stall_check)
    assert L.iris_wait_probe(3, 0) == _lib.IRIS_ESTALL  # left for those who ask
    asks = [generate, serving.stall_check]
    for ask in asks if first == "session" else reversed(asks):
        assert stalled(ask)
    for ask in asks:
        assert not stalled(ask)
    assert generate() == want
    dm.close()
    assert L.iris_wait_probe(4, 1) == _lib.IRIS_EINVAL
