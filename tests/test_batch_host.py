"""Host side of the serving-step operators without a GPU: what they ask of the CUDA runtime, over a stand-in for it
(fake_device)."""
import pytest

import fake_device

pytestmark = pytest.mark.skipif(fake_device.nvcc() is None, reason="no nvcc")


@pytest.fixture
def dev(kvx):
    return fake_device.Device(kvx)


BESIDE = dict(batch=64, hq=32, hkv=8, dim=128, prefix_len=32768, max_len=1024)  # prefix and tails share the device


@pytest.mark.parametrize("again", [BESIDE, dict(BESIDE, batch=60)])
def test_runs_after_a_failed_call(dev, kvx, again):
    """A call whose combine pass was not launched does not leave the next one a used-up counter of runs."""
    _, h = dev.create(64, 32, 8, 128)
    assert dev.attend(h, **BESIDE) == kvx.KVX_OK
    assert [(x.kind, x.shared_runs, x.counter) for x in dev.launches()[:2]] == [("prefix", 1, 0), ("stream", 1, 0)]
    dev.lib.fake_fail_launch(2)
    assert dev.attend(h, **BESIDE) == kvx.KVX_ERR_CUDA
    assert [x.kind for x in dev.launches()] == ["prefix", "stream"]
    assert dev.attend(h, 64, 32, 8, 128, max_len=100) == kvx.KVX_OK  # (takes no runs from the counter)
    dev.launches()
    assert dev.attend(h, **again) == kvx.KVX_OK
    assert [(x.kind, x.shared_runs, x.counter) for x in dev.launches()[:2]] == [("prefix", 1, 0), ("stream", 1, 0)]
    dev.lib.kvx_batch_destroy(h)
