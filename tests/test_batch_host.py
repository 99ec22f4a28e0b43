"""Host side of the serving-step operators without a GPU: what they ask of the CUDA runtime, over a stand-in for it
(fake_device)."""
import math
import random

import pytest

import fake_device
import long_cases

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


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_shared_memory_is_allowed_on_every_device(dev, kvx, dim, dtype):
    """A kernel's limit of shared memory belongs to a device: a handle on another one launches as well."""
    for ordinal in (0, 1, 2):
        dev.lib.fake_set_device(ordinal)
        rc, h = dev.create(2048, 8, 2, dim, dtype)
        assert rc == kvx.KVX_OK
        coded = [dev.lib.fake_prefix(2, dim, 5000)] if dtype == 0 else []
        for prefix in [dict(prefix_len=1000), dict(prefix_len=1000, page_tokens=5), {}] + [dict(coded=p) for p in coded]:
            assert dev.attend(h, 2048, 8, 2, dim, max_len=100, **prefix) == kvx.KVX_OK, (ordinal, prefix, dev.lib.fake_last_error())
        assert {x.device for x in dev.launches()} == {ordinal}
        for p in coded:
            dev.lib.fake_prefix_free(p)
        dev.lib.kvx_batch_destroy(h)


def test_a_refused_limit_is_not_remembered(dev, kvx):
    before = dev.lib.fake_live_allocations()
    for n in range(3):
        dev.lib.fake_fail_attribute(n)
        rc, h = dev.create(4, 8, 2, 64)
        assert rc == kvx.KVX_ERR_CUDA and not h.value and dev.lib.fake_live_allocations() == before
    rc, h = dev.create(4, 8, 2, 64)
    assert rc == kvx.KVX_OK and dev.attend(h, 4, 8, 2, 64, 1000, 100) == kvx.KVX_OK
    dev.lib.kvx_batch_destroy(h)


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_older_kernels_launch_on_every_device(dev, kvx, dim):
    """The decode attention kernel of every kind of plan and the encoder, whose limits are raised where they are
    launched; a failure is not kept."""
    calls = [lambda: dev.lib.fake_decode_attention(dim, 1, 0), lambda: dev.lib.fake_decode_attention(dim, 0, 1),
             lambda: dev.lib.fake_decode_attention(dim, 0, 0), lambda: dev.lib.fake_encode(dim)]
    for ordinal in (0, 1, 5):
        dev.lib.fake_set_device(ordinal)
        assert [c() for c in calls] == [0, 0, 0, 0], ordinal
        assert [x.device for x in dev.launches()] == [ordinal] * 4
        assert [c() for c in calls] == [0, 0, 0, 0]
        dev.launches()
    dev.lib.fake_set_device(10 + dim // 32)  # (no other test uses it)
    for c in calls[:3]:
        dev.lib.fake_fail_attribute(0)
        assert c() != 0 and not dev.launches()
        assert c() == 0 and len(dev.launches()) == 1


def test_a_batch_belongs_to_its_device(dev, kvx):
    """Its calls are refused, with nothing launched, while another device is current; so is another device's prefix."""
    dev.lib.fake_set_device(1)
    _, h = dev.create(8, 8, 2, 64)
    calls = [lambda: dev.attend(h, 8, 8, 2, 64, 1000, 100), lambda: dev.rotate(h, 5, 8, 64), lambda: dev.append(h, 5, 2, 64),
             lambda: dev.lib.kvx_batch_check(h)]
    assert [c() for c in calls] == [kvx.KVX_OK] * 4
    assert {x.device for x in dev.launches()} == {1}
    dev.lib.fake_set_device(0)
    for c in calls:
        assert c() == kvx.KVX_ERR_INVALID_ARGUMENT
        assert dev.lib.fake_last_error().endswith(b"the batch was made on device 1, and device 0 is current")
    p = dev.lib.fake_prefix(2, 64, 500)  # (made on device 0)
    dev.lib.fake_set_device(1)
    assert dev.attend(h, 8, 8, 2, 64, 0, 100, coded=p) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert b"another device" in dev.lib.fake_last_error() and not dev.launches()
    dev.lib.fake_prefix_free(p)
    dev.lib.kvx_batch_destroy(h)


def test_a_success_clears_the_last_error(dev, kvx):
    _, h = dev.create(8, 8, 2, 64)
    for call in (lambda: dev.attend(h, 8, 8, 2, 64, 1000, 100), lambda: dev.attend(h, 0, 8, 2, 64), lambda: dev.rotate(h, 5, 8, 64),
                 lambda: dev.rotate(h, 0, 8, 64), lambda: dev.append(h, 5, 2, 64), lambda: dev.append(h, 0, 2, 64),
                 lambda: dev.lib.kvx_batch_wait_limit(h, 5), lambda: dev.lib.kvx_batch_check(h)):
        dev.lib.fake_set_error(b"an earlier call's")
        assert call() == kvx.KVX_OK and dev.lib.fake_last_error() == b""
    dev.lib.kvx_batch_destroy(h)


def test_long_cases_have_long_items(dev, kvx):
    """The GPU test of the prefix kernel's steady state has items of as many tiles as it is meant to."""
    for hq, hkv, dim, batch, prefix, page, dtype in long_cases.CASES:
        rc, h = dev.create(batch, hq, hkv, dim, int(dtype == "fp16"))
        coded = dev.lib.fake_prefix(hkv, dim, prefix) if page == 0 else None
        paged = {} if page == 0 else dict(prefix_len=prefix, page_tokens=page)
        assert rc == kvx.KVX_OK and dev.attend(h, batch, hq, hkv, dim, max_len=5, coded=coded, **paged) == kvx.KVX_OK
        x = dev.launches()[0]
        assert x.kind == "prefix" and x.split_tiles >= long_cases.LEAST_TILES
        dev.lib.kvx_batch_destroy(h)
        if coded:
            dev.lib.fake_prefix_free(coded)
    loaders = {(c[2], c[5] == 0, c[5] % 8 == 0, c[6]) for c in long_cases.CASES}
    for dim in (32, 64, 128, 256):
        assert (dim, True, True, "bf16") in loaders
        assert {t for d, coded, tma, t in loaders if d == dim and not coded and not tma} == {"bf16", "fp16"}
        assert any(d == dim and not coded and tma for d, coded, tma, t in loaders)


def test_every_cut_covers_its_prefix_and_fits_the_scratch(dev, kvx):
    """Random layouts and lengths over the accepted ranges: the items cover every tile once, and the partial states fit."""
    rng = random.Random(5)

    def upto(n):
        return int(math.exp(rng.uniform(0.0, math.log(n))))

    for _ in range(400):
        hkv, group, dim, dtype = upto(200), upto(40), rng.choice([32, 64, 128, 256]), rng.choice([0, 1])
        most = upto(min(2048, max(1, 60000 // (hkv * group))))
        hq = hkv * group
        rc, h = dev.create(most, hq, hkv, dim, dtype)
        assert rc == kvx.KVX_OK
        for _ in range(6):
            batch, prefix, tail, page = upto(most), upto(1 << 21) if rng.random() < 0.8 else 0, upto(1 << 17) - 1, rng.choice([1, 7, 16, 64])
            coded = dev.lib.fake_prefix(hkv, dim, prefix) if prefix and dtype == 0 and rng.random() < 0.4 else None
            rc = dev.attend(h, batch, hq, hkv, dim, 0 if coded else prefix, tail, page, coded)
            assert rc == kvx.KVX_OK, (hq, hkv, dim, most, batch, prefix, tail, page, dev.lib.fake_last_error())
            ran = dev.launches()
            kinds = [x.kind for x in ran]
            streamed = tail > 0 or (prefix > 0 and coded is None and batch * group <= 8)
            tensor = prefix > 0 and (coded is not None or batch * group > 8)
            assert kinds == ["prefix"] * tensor + ["stream"] * streamed + ["combine"]
            if tensor:
                x = ran[0]
                assert x.prefix_tiles == -(-prefix // 64) and x.row_groups == -(-batch * group // 128)
                assert (x.n_split - 1) * x.split_tiles < x.prefix_tiles <= x.n_split * x.split_tiles
                assert x.grid == hkv * x.n_split * x.row_groups
            if coded:
                dev.lib.fake_prefix_free(coded)
        dev.lib.kvx_batch_destroy(h)
