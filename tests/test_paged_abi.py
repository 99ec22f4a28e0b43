"""CPU checks of the serving-step entry points: argument errors come before any CUDA call."""
import ctypes as C

import pytest


@pytest.mark.parametrize("args", [(0, 4, 2, 64, 0), (70000, 4, 2, 64, 0), (1, 4, 3, 64, 0), (1, 0, 1, 64, 0),
                                  (1, 4, 0, 64, 0), (1, 4, 2, 63, 0), (1, 4, 2, 258, 0), (1, 4, 2, 0, 0), (1, 4, 2, 64, 2)])
def test_batch_create_refuses(kvx, args):
    h = C.c_void_p()
    assert kvx._batch_create(*args, C.byref(h)) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert b"kvx_batch_create" in kvx._last_error() and not h.value


def test_null_handles(kvx):
    v = bytes(kvx.kvx_view(16, 64, 64))
    r = bytes(kvx.kvx_rope(16, 16, 16, None, 0, 1, 64, 1, 0))
    p = bytes(kvx.kvx_pages(16, 16, 64, 64, 64, 1, 1))
    assert kvx._batch_rotate(None, v, v, 1, 1, r, 0, None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_append(None, None, v, v, None, 1, None, 16, p, None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_attend(None, bytes(kvx.kvx_attend()), None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_check(None) == kvx.KVX_ERR_INVALID_ARGUMENT
    kvx._batch_destroy(None)


def test_host_tensors_are_refused(kvx):
    import torch
    x = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kvx.Pages(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        kvx.Rope(torch.zeros((4, 32)), torch.zeros((4, 32)))
    with pytest.raises(ValueError, match="dtype"):
        kvx.Batch(1, 1, 1, 64, dtype="fp32")


@pytest.mark.parametrize("args", [(2049, 8, 2, 64, 0), (1, 65538, 2, 64, 0)])
def test_batch_create_refuses_what_it_cannot_count(kvx, args):
    """More sequences or heads than the streaming kernel's lists and the grids are for."""
    h = C.c_void_p()
    assert kvx._batch_create(*args, C.byref(h)) == kvx.KVX_ERR_INVALID_ARGUMENT and not h.value


def test_wait_limit_of_no_batch(kvx):
    assert kvx._batch_wait_limit(None, 1) == kvx.KVX_ERR_INVALID_ARGUMENT
